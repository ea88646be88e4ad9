"""The paged cache's C entry points and index arithmetic, on the CPU: refusals
(every call here returns before anything is enqueued), the Rust mirror, and the
kernels' index functions walked over lengths and tables of any content."""
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

import llmoxide_amd as lmx
from llmoxide_amd import paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "lmx", "paged.h")
RUST = os.path.join(ROOT, "rust", "llmoxide-hip-ffi", "src", "paged.rs")
FAKE = 0x100000  # never dereferenced: validation fails first
FAR = FAKE + (1 << 32)
S = lmx.Status


def header():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_header_compiles_as_c_and_cxx(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "lmx/paged.h"\nint main(void){lmxp_pool p; return sizeof p == 0;}\n')
    for cc, extra in (("gcc", ["-std=c99"]), ("g++", ["-x", "c++", "-std=c++17"])):
        r = subprocess.run([cc, *extra, "-fsyntax-only", "-Wall", "-Werror", "-I",
                            os.path.join(ROOT, "include"), str(src)], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr


def test_library_exports_what_the_header_declares():
    names = set(re.findall(r"\b(lmxp_\w+)\s*\(", header()))
    assert names == set(paged.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", lmx.LIB_PATH], capture_output=True, text=True).stdout
    assert set(re.findall(r"\bT (lmxp_\w+)", out)) == names


C_TYPES = {"uint32_t": "u32", "float": "f32", "int32_t": "i32", "void": "c_void", "lmx_dtype": "i32",
           "lmx_status": "i32", "lmx_stream": "HipStream", "size_t": "usize"}


def to_rust(ctype):
    const = "const" in ctype
    words = [w for w in re.findall(r"\w+|\*", ctype) if w != "const"]
    base, stars = words[0], words.count("*")
    t = C_TYPES.get(base) or "".join(p.capitalize() for p in base.split("_"))
    assert stars <= 1, ctype
    return ("*const " if const else "*mut ") + t if stars else t


def test_rust_mirror_matches():
    src = re.sub(r"//[^\n]*", "", open(RUST).read())
    structs = {n: re.findall(r"pub (\w+): ([^,]+),", b) for n, b in re.findall(r"pub struct (\w+) \{(.*?)\}", src, flags=re.S)}
    for body, name in re.findall(r"typedef struct \{(.*?)\}\s*(\w+);", header(), flags=re.S):
        want = []
        for decl in body.split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            kind, names = re.match(r"^((?:const )?\w+ \*?)(.*)$", decl).groups()
            want += [(n.strip(" *"), to_rust(kind)) for n in names.split(",")]
        rust = "".join(p.capitalize() for p in name.split("_"))
        assert structs[rust] == want, (rust, structs.get(rust), want)
    fns = {}
    for name, args, ret in re.findall(r"pub fn (lmxp_\w+)\((.*?)\)\s*->\s*([^;]+);", src, flags=re.S):
        fns[name] = ([tuple(x.strip() for x in a.split(":")) for a in args.split(",") if a.strip()], ret.strip())
    for ret, name, args in re.findall(r"^(\w+) (lmxp_\w+)\(([^;]*?)\);", header(), flags=re.M | re.S):
        want = []
        for a in " ".join(args.split()).split(","):
            kind, n = re.match(r"^(.*?)(\w+)$", a.strip()).groups()
            want.append((n, to_rust(kind)))
        assert fns[name] == (want, to_rust(ret)), (name, fns.get(name), want)
    assert len(fns) == len(paged.SIGNATURES)
    for k, v in re.findall(r"\b(LMXP_\w+)\s*=\s*(\d+)", header()):
        assert re.search(rf"pub const {k}: u32 = {v};", src), k


# ----------------------------------------------------------------- refusals --
def pool(**kw):
    d = dict(n_pages=8, page_size=16, n_kv_heads=2, head_dim=128, store=paged.STORE_F16, k=FAKE, v=FAKE,
             k_scale=None, v_scale=None)
    d.update(kw)
    return paged.PoolDesc(**d)


def batch(**kw):
    d = dict(n_seq=2, n_tokens=4, max_new=3, max_ctx=64, table_stride=4, cu=FAKE, ctx_lens=FAKE, page_table=FAKE)
    d.update(kw)
    return paged.BatchDesc(**d)


def append(p=None, b=None, k=FAKE, v=FAKE, dt=lmx.F32, stride=0):
    return paged.paged_lib().lmxp_append(ctypes.byref(p or pool()), ctypes.byref(b or batch()), k, v, dt, stride, None)


def read(p=None, b=None, k=FAKE, v=FAKE, dt=lmx.F32, stride=0):
    return paged.paged_lib().lmxp_read(ctypes.byref(p or pool()), ctypes.byref(b or batch()), k, v, dt, stride, None)


def prologue(p=None, b=None, q=FAKE, k=FAKE, v=FAKE, qg=None, kg=None, rf=None, out=FAR, dt=lmx.F32, **kw):
    d = dict(n_heads=4, n_rot=128, v_norm=0, q_head_stride=0, q_row_stride=0, kv_row_stride=0, rms_eps=1e-6,
             rope_base=1e6)
    d.update(kw)
    return paged.paged_lib().lmxp_prologue(ctypes.byref(p or pool()), ctypes.byref(b or batch()),
                                           ctypes.byref(paged.PagedPrologueDesc(**d)), q, k, v, qg, kg, rf, out,
                                           dt, None)


def attn(p=None, b=None, q=FAKE, out=FAR, dt=lmx.F32, ws=None, ws_bytes=0, **kw):
    d = dict(n_heads=4, window=0, q_head_stride=0, q_row_stride=0, scale=0.1)
    d.update(kw)
    return paged.paged_lib().lmxp_attn(ctypes.byref(p or pool()), ctypes.byref(b or batch()),
                                       ctypes.byref(paged.PagedAttnDesc(**d)), q, dt, out, ws, ws_bytes, None)


BAD_POOLS = [
    (dict(head_dim=96), S.E_UNSUPPORTED), (dict(head_dim=0), S.E_UNSUPPORTED), (dict(page_size=8), S.E_UNSUPPORTED),
    (dict(page_size=48), S.E_UNSUPPORTED), (dict(page_size=512), S.E_UNSUPPORTED), (dict(store=0), S.E_UNSUPPORTED),
    (dict(store=3), S.E_UNSUPPORTED), (dict(n_kv_heads=0), S.E_SHAPE), (dict(n_pages=0), S.E_SHAPE),
    (dict(k=None), S.E_NULL), (dict(v=None), S.E_NULL), (dict(k=FAKE + 8), S.E_ALIGN), (dict(v=FAKE + 2), S.E_ALIGN),
    (dict(store=paged.STORE_I8), S.E_NULL),
    (dict(store=paged.STORE_I8, k_scale=FAKE, v_scale=FAKE + 4), S.E_ALIGN),
]
BAD_BATCHES = [
    (dict(n_seq=0), S.E_SHAPE), (dict(n_tokens=0), S.E_SHAPE), (dict(max_new=0), S.E_SHAPE),
    (dict(max_new=5), S.E_SHAPE), (dict(max_ctx=0), S.E_SHAPE), (dict(max_ctx=65), S.E_CONTEXT),
    (dict(table_stride=0), S.E_SHAPE), (dict(cu=None), S.E_NULL), (dict(ctx_lens=None), S.E_NULL),
    (dict(page_table=None), S.E_NULL), (dict(cu=FAKE + 2), S.E_ALIGN), (dict(page_table=FAKE + 1), S.E_ALIGN),
    (dict(max_ctx=1 << 30, table_stride=1 << 29), S.E_CONTEXT),
]


@pytest.mark.parametrize("call", [append, read, prologue, attn])
@pytest.mark.parametrize("kw,code", BAD_POOLS)
def test_bad_pools_are_refused(call, kw, code):
    assert call(p=pool(**kw)) == code


@pytest.mark.parametrize("call", [append, read, prologue, attn])
@pytest.mark.parametrize("kw,code", BAD_BATCHES)
def test_bad_batches_are_refused(call, kw, code):
    assert call(b=batch(**kw)) == code


@pytest.mark.parametrize("call", [append, read])
@pytest.mark.parametrize("kw,code", [
    (dict(k=None, v=None), S.E_NULL), (dict(dt=7), S.E_UNSUPPORTED), (dict(stride=255), S.E_SHAPE),
    (dict(stride=258), S.E_SHAPE), (dict(k=FAKE + 8), S.E_ALIGN), (dict(dt=lmx.F16, v=FAKE + 4), S.E_ALIGN),
])
def test_bad_rows_are_refused(call, kw, code):
    assert call(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), S.E_NULL), (dict(k=None), S.E_NULL), (dict(v=None), S.E_NULL), (dict(out=None), S.E_NULL),
    (dict(dt=9), S.E_UNSUPPORTED), (dict(n_rot=130), S.E_SHAPE), (dict(n_rot=5), S.E_SHAPE), (dict(v_norm=2), S.E_SHAPE),
    (dict(rope_base=0.0), S.E_SHAPE), (dict(rope_base=float("inf")), S.E_SHAPE), (dict(rms_eps=-1.0), S.E_SHAPE),
    (dict(rms_eps=float("nan")), S.E_SHAPE), (dict(n_heads=0), S.E_SHAPE), (dict(q_head_stride=64), S.E_SHAPE),
    (dict(q_head_stride=130), S.E_SHAPE), (dict(q_row_stride=256), S.E_SHAPE), (dict(kv_row_stride=128), S.E_SHAPE),
    (dict(q=FAKE + 4), S.E_ALIGN), (dict(qg=FAKE + 4), S.E_ALIGN), (dict(out=FAR + 8), S.E_ALIGN),
    (dict(out=FAKE + 1024), S.E_SHAPE),                       # into q's rows
    (dict(out=FAKE, dt=lmx.F16), S.E_SHAPE),                  # in place, but another type
    (dict(out=FAKE, q_head_stride=256), S.E_SHAPE),           # in place, but strided
    (dict(q=FAR, out=FAKE + 512), S.E_SHAPE),                 # into k_new / v_new
])
def test_bad_prologues_are_refused(kw, code):
    assert prologue(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), S.E_NULL), (dict(out=None), S.E_NULL), (dict(dt=2), S.E_UNSUPPORTED), (dict(n_heads=3), S.E_SHAPE),
    (dict(n_heads=0), S.E_SHAPE), (dict(scale=float("nan")), S.E_SHAPE), (dict(scale=float("inf")), S.E_SHAPE),
    (dict(q_head_stride=132), S.E_SHAPE), (dict(q_head_stride=120), S.E_SHAPE), (dict(q_row_stride=504), S.E_SHAPE),
    (dict(window=1 << 30), S.E_SHAPE), (dict(q=FAKE + 8), S.E_ALIGN), (dict(out=FAR + 8), S.E_ALIGN),
    (dict(out=FAKE), S.E_SHAPE), (dict(out=FAKE + 4 * 512 * 4 - 16), S.E_SHAPE),
])
def test_bad_attention_calls_are_refused(kw, code):
    assert attn(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(), S.E_WORKSPACE), (dict(ws=FAKE, ws_bytes=16), S.E_WORKSPACE), (dict(ws=FAKE + 8, ws_bytes=1 << 30), S.E_ALIGN),
])
def test_a_split_attention_needs_its_workspace(kw, code):
    """Contexts long enough to be cut between workgroups."""
    assert attn(b=batch(max_ctx=4096, table_stride=256), **kw) == code


def test_null_descriptions_are_refused():
    L = paged.paged_lib()
    p, b = ctypes.byref(pool()), ctypes.byref(batch())
    assert L.lmxp_append(None, b, FAKE, FAKE, 0, 0, None) == S.E_NULL
    assert L.lmxp_append(p, None, FAKE, FAKE, 0, 0, None) == S.E_NULL
    assert L.lmxp_prologue(p, b, None, FAKE, FAKE, FAKE, None, None, None, FAR, 0, None) == S.E_NULL
    assert L.lmxp_attn(p, b, None, FAKE, 0, FAR, None, 0, None) == S.E_NULL
    assert L.lmxp_attn_workspace_bytes(None, b, None) == 0
    assert L.lmxp_attn_workspace_bytes(p, b, None) == 0


def test_counts_that_pass_32_bits_are_refused():
    assert attn(p=pool(n_pages=1 << 20), b=batch(n_tokens=1 << 27, max_new=1 << 27, max_ctx=1 << 28,
                                                 table_stride=1 << 25)) == S.E_SHAPE


def test_launches_too_large_to_name_are_refused():
    """2^24 workgroups and more, or 2^16 heads side by side."""
    many = batch(n_seq=1 << 20, n_tokens=1 << 22, max_new=4)
    assert append(p=pool(n_kv_heads=256), b=many) == S.E_SHAPE              # 2^22 rows x 512 heads / 16 a workgroup
    assert prologue(p=pool(n_kv_heads=256), b=many, n_heads=256, out=1 << 44) == S.E_SHAPE
    long = batch(n_tokens=1 << 28, max_new=1 << 28)
    assert append(p=pool(head_dim=512), b=long) == S.E_SHAPE                # 16 rows a workgroup
    assert read(p=pool(head_dim=512), b=long) == S.E_SHAPE
    assert prologue(b=batch(n_tokens=8, max_new=8), n_heads=65536, out=1 << 44) == S.E_SHAPE
    wide = batch(n_seq=1 << 20, n_tokens=1 << 20, max_new=1, max_ctx=4096, table_stride=256)
    assert attn(p=pool(n_kv_heads=512), b=wide, n_heads=512, out=1 << 44) == S.E_SHAPE
    d = paged.PagedAttnDesc(n_heads=512, window=0, q_head_stride=0, q_row_stride=0, scale=0.1)
    assert paged.paged_lib().lmxp_attn_workspace_bytes(ctypes.byref(pool(n_kv_heads=512)), ctypes.byref(wide),
                                                       ctypes.byref(d)) == 0


# ---------------------------------------------------------- index arithmetic --
WALK = r"""
#include "paged_index.hpp"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace lmx;
static uint32_t st = 12345;
static uint32_t rnd() { st = st * 1664525u + 1013904223u; return st >> 8; }
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    for (int round = 0; round < 4000; ++round) {
        const bool garbage = round & 1;
        PagedGeom g{};
        g.n_seq = 1 + rnd() % 70;
        g.ps_log2 = 4 + rnd() % 5;
        g.table_stride = 1 + rnd() % 40;
        g.n_pages = 1 + rnd() % 500;
        g.max_ctx = 1 + rnd() % (g.table_stride << g.ps_log2);
        g.Hkv = 1 + rnd() % 8;
        g.G = 1 + rnd() % 9;
        g.window = rnd() % 3 ? 0 : 1 + rnd() % 300;
        std::vector<int> cu(g.n_seq + 1), ctx(g.n_seq);
        int at = 0;
        for (int b = 0; b < g.n_seq; ++b) {
            ctx[b] = rnd() % (g.max_ctx + 1);
            cu[b] = at;
            at += rnd() % 4 ? (ctx[b] ? 1 : 0) : (int)(rnd() % (ctx[b] + 1));
        }
        cu[g.n_seq] = at;
        g.n_tokens = at ? at : 1;
        if (garbage)
            for (int b = 0; b <= g.n_seq; ++b) {
                if (rnd() % 3 == 0) cu[b] = (int)(rnd() << 8 ^ rnd());
                if (b < g.n_seq && rnd() % 3 == 0) ctx[b] = (int)(rnd() << 8 ^ rnd());
            }
        for (int bm : {16, 128}) {
            const int target = 512, least = 2;
            double work = 0;
            int64_t items = 0;
            for (int pass = 0; pass < 2; ++pass) {
                const int per = pass ? units_per_split((float)work, target, least) : 0;
                for (int b = 0; b < g.n_seq; ++b) {
                    const PagedSeq s = paged_seq(g, cu[b], cu[b + 1], ctx[b]);
                    CHECK(s.row0 >= 0 && s.n >= 0 && s.row0 + s.n <= g.n_tokens);
                    CHECK(s.ctx >= 0 && s.ctx <= g.max_ctx);
                    const SeqWork w = seq_work(g, s, bm);
                    CHECK(w.lo >= 0 && w.lo % kUnit == 0 && w.lo <= s.ctx && w.units >= 0);
                    CHECK(w.lo + w.units * kUnit >= s.ctx);
                    if (!pass) { work += (double)w.rt * w.units * g.Hkv; continue; }
                    const int n = seq_splits(w, per);
                    CHECK(n >= 1 && (int64_t)n * per >= w.units && (int64_t)(n - 1) * per < (w.units ? w.units : 1));
                    items += (int64_t)w.rt * g.Hkv * n;
                    for (int i = 0; i < 40; ++i) {
                        const int pos = garbage ? (int)(rnd() << 8 ^ rnd()) : (int)(rnd() % (w.lo + w.units * kUnit + 1));
                        const int e = paged_entry(g, pos);
                        CHECK(e >= -1 && e < g.table_stride);
                    }
                }
            }
            if (!garbage) {
                CHECK(items <= row_tiles_bound(g, bm) * g.Hkv + target);
                int64_t tiles = 0;
                for (int b = 0; b < g.n_seq; ++b) tiles += seq_work(g, paged_seq(g, cu[b], cu[b + 1], ctx[b]), bm).rt;
                CHECK(tiles <= row_tiles_bound(g, bm) && (at == 0 || tiles >= row_tiles_least(g, bm)));
            }
        }
        for (int log2_r = 4; log2_r <= 6; ++log2_r) {  // row blocks: every row once, cut at whole granules
            int64_t blocks = 0;
            for (int b = 0; b < g.n_seq; ++b) {
                const PagedSeq s = paged_seq(g, cu[b], cu[b + 1], ctx[b]);
                const int n = row_blocks(s, log2_r);
                int next = 0;
                for (int i = 0; i < n; ++i) {
                    const RowBlock r = row_block(s, i, log2_r);
                    CHECK(r.first == next && r.count > 0 && r.count <= 1 << log2_r);
                    CHECK(i == 0 || ((s.ctx - s.n + r.first) & ((1 << log2_r) - 1)) == 0);
                    next += r.count;
                    if (garbage && i > 64) { next = s.n; break; }
                }
                CHECK(next == s.n);
                blocks += n;
            }
            if (!garbage) CHECK(blocks <= row_blocks_bound(g, log2_r));
        }
        for (int i = 0; i < 50; ++i) {
            const int page = paged_page(g, (int)(rnd() << 8 ^ rnd()));
            CHECK(page >= -1 && page < g.n_pages);
        }
        CHECK(paged_page(g, -1) == -1 && paged_page(g, g.n_pages) == -1 && paged_page(g, g.n_pages - 1) == g.n_pages - 1);
    }
    printf("ok\n");
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_index_arithmetic_stays_in_range_whatever_the_tables_hold(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(WALK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(ROOT, "llmoxide_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.stdout == "ok\n", r.stdout + r.stderr


# ------------------------------------------------------------------- oracle --
def test_oracle_quantise():
    from tests.paged_oracle import quantise
    x = np.zeros(64, np.float32)
    assert quantise(x)[1] == 0
    x[3] = 127.0
    x[4], x[5], x[6] = 0.5, 1.5, -2.5  # ties at scale 1
    q, s = quantise(x)
    assert s == 1 and list(q[3:7]) == [127, 0, 2, -2]
    x[7] = np.inf
    q, s = quantise(x)
    assert np.isnan(s) and not q.any()


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("window", [0, 9])
def test_oracle_attention_is_the_textbooks(store, window):
    """Each sequence's pages laid out side by side, against the contiguous form."""
    from oracle import textbook
    from tests import paged_oracle as po
    c = po.PagedCase(3, new=[1, 5, 0, 17], ctx=[40, 5, 9, 30], page=16, kv=2, hd=64, store=store)
    q = np.random.default_rng(4).standard_normal((c.tokens, 6, 64))
    got = po.attend(c, q, heads=6, window=window)[0]
    for b, (n, ctx) in enumerate(zip(c.new, c.ctx)):
        if not n:
            continue
        kv = [[c.held(b, h, p) for h in range(2)] for p in range(ctx)]
        k = np.array([[x[0] for x in row] for row in kv])
        v = np.array([[x[1] for x in row] for row in kv])
        rows = slice(int(c.cu[b]), int(c.cu[b]) + n)
        want = textbook.attention(q[rows], k, v, n_heads=6, n_kv_heads=2, head_dim=64, base_pos=ctx - n, window=window)
        assert np.abs(got[rows].reshape(n, -1) - want).max() < 1e-12


@pytest.mark.parametrize("n_rot", [64, 32])
def test_oracle_rotation_is_the_textbooks(n_rot):
    from oracle import textbook
    from tests.paged_oracle import rope_norm
    x = np.random.default_rng(5).standard_normal(64)
    want = x.copy()
    want[:n_rot] = textbook.rope_neox(x[:n_rot], 77, 1e4)
    assert np.abs(rope_norm(x, None, 77, n_rot=n_rot, eps=0, base=1e4) - want).max() < 1e-12
    gain = np.linspace(0.5, 2, 64)
    want = x / np.sqrt((x * x).mean() + 1e-6) * gain
    assert np.abs(rope_norm(x, gain, 0, n_rot=n_rot, eps=1e-6, base=1e4) - want).max() < 1e-12


@pytest.mark.parametrize("store", ["f16", "i8"])
def test_oracle_append_is_read_where_it_belongs(store):
    from tests import paged_oracle as po
    c = po.PagedCase(6, new=[3, 0, 20], ctx=[18, 4, 20], page=16, kv=2, hd=64, store=store)
    before = [x.copy() for x in (c.k, c.v)]
    x = np.random.default_rng(7).standard_normal((2, c.tokens, 2, 64)).astype(np.float32)
    c.k, c.v, c.k_scale, c.v_scale = po.append(c, x[0], x[1])
    for row, b, pos, at in c.row_places():
        for h in range(2):
            for got, want in zip(c.held(b, h, pos), x[:, row, h]):
                # half a step of f16 at 4, or of amax / 127
                assert np.abs(got - want).max() <= (2.0 ** -9 if store == "f16" else 0.501 * np.abs(want).max() / 127)
    own = {c.place(b, p) for row, b, p, _ in c.row_places()}
    for now, was, slot in ((c.k, before[0], 2), (c.v, before[1], 3)):
        off = np.moveaxis(now != was, slot, 1).any(axis=(2, 3))
        assert {tuple(int(y) for y in t) for t in np.argwhere(off)} <= own


def test_rows_that_share_memory_are_refused():
    """A row stride of 0 means dense to the library: broadcast rows must not reach it."""
    torch = pytest.importorskip("torch")
    x = torch.zeros(1, 64)
    assert paged._rows(torch.zeros(4, 64), 4, 64, "q") == 0 and paged._rows(x, 1, 64, "q") == 0
    assert paged._rows(torch.zeros(4, 100)[:, 8:72], 4, 64, "q") == 100
    for bad in (x.expand(4, 64), torch.zeros(200).as_strided((4, 64), (32, 1)), torch.zeros(4, 128)[:, ::2],
                torch.empty_strided((2, 64), (1 << 32, 1), device="meta")):
        with pytest.raises(ValueError):
            paged._rows(bad, *bad.shape, "q")
