"""Calls on a stream beside the current one, while the current one still uses memory
that it has freed: the call's results and workspaces are not made of it."""
import numpy as np
import pytest

from tests import paged_oracle as po

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llmoxide_amd as lmx  # noqa: E402
from tests.test_gpu_paged import gpu, on_gpu, rows, say  # noqa: E402
from tests.test_gpu_spec import ints, verify_case  # noqa: E402


def paged_calls():
    c = po.PagedCase(120, new=[40, 9], ctx=[3000, 700], page=16, kv=2, hd=128)
    cache, batch = on_gpu(c)
    q, k, v = (gpu(rows(c, 121 + i, h).reshape(c.tokens, -1)) for i, h in enumerate((8, 2, 2)))
    parent = ints(np.concatenate([np.arange(-1, n - 1) for n in c.new]))
    seen = lmx.spec_tree(parent, batch).seen
    t = verify_case(122, [9, 30], 50000, "tree", "sampled")
    args = [gpu(t[x]) for x in ("p", "tok", "u", "r", "cu")]
    kw = dict(max_new=30, parent=ints(np.concatenate(t["trees"])), q=gpu(t["q"]))
    tables = [lmx.PageTables.empty(60, page_size=16, n_seq=2, entries=30) for _ in range(2)]
    lens, new = ints([100, 3]), ints([30, 19])
    return {
        "paged_read": lambda s: lmx.paged_read(cache, batch, stream=s),
        "paged_prologue": lambda s: [lmx.paged_prologue(q, k, v, cache, batch, n_heads=8, stream=s)],
        "paged_attention": lambda s: [lmx.paged_attention(q, cache, batch, n_heads=8, stream=s)],
        "spec_plan": lambda s: lmx.spec_plan(tables[s is None], lens, new, n_tokens=49, stream=s),
        "spec_tree": lambda s: lmx.spec_tree(parent, batch, stream=s),
        "spec_prologue": lambda s: [lmx.spec_prologue(q, k, v, cache, batch, n_heads=8, q_dtype=d, stream=s)
                                    for d in (None, torch.float16)],
        "spec_attention": lambda s: [lmx.spec_attention(q, cache, batch, seen, n_heads=8, stream=s)],
        "spec_verify": lambda s: lmx.spec_verify(*args, stream=s, **kw),
    }


def other_calls():
    g = torch.Generator("cuda").manual_seed(5)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)
    q, one = randn(70, 8 * 128), randn(2, 8 * 128)
    k, v = randn(3000, 256, dtype=torch.float16), randn(3000, 256, dtype=torch.float16)
    caches = lmx.BatchedCaches([k, v], [v, k])
    ctx = ints([2900, 77])
    kw = dict(n_heads=8, n_kv_heads=2, head_dim=128)
    x, taps, state = randn(50, 512), randn(512, 4), randn(3, 512)
    conv, alpha, beta = randn(128, 512), randn(128, 2), randn(128, 2)
    delta, a, bias = randn(2, 128, 128) * 0.01, randn(2), randn(2)
    dkw = dict(n_vh=2, n_kh=1, s_dim=128)
    w, y = torch.randint(0, 50, (256 * 34,), generator=g, device="cuda", dtype=torch.uint8), randn(3, 256)
    return {
        "attention": lambda s: [lmx.attention(q, k, v, base_pos=2500, stream=s, **kw)],
        "attention of one": lambda s: [lmx.attention(one[:1], k, v, base_pos=2500, stream=s, **kw)],
        "attention_decode_batched": lambda s: [lmx.attention_decode_batched(one, caches, ctx, max_ctx=2900, stream=s, **kw)],
        "delta_recur": lambda s: [lmx.delta_recur(conv, alpha, beta, delta.clone() if s is None else delta, a, bias, stream=s, **dkw)],
        "delta_front": lambda s: [lmx.delta_front(x, taps, state.clone() if s is None else state, key_dim=128, s_dim=128, stream=s)],
        "matvec": lambda s: [lmx.matvec(w[:256 * 34 // 32 * 32], y, qtype="q8_0", rows=32, in_dim=256, stream=s)],
    }


@pytest.mark.parametrize("calls", [paged_calls, other_calls])
def test_results_on_a_side_stream_leave_what_the_current_one_still_reads(calls):
    side = torch.cuda.Stream()
    for name, call in calls().items():
        say("side stream", name)
        want = [x.clone() for x in call(None) if x is not None]
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        # what the current stream reads behind a long kernel, and has given back by then
        sizes = [x.numel() * x.element_size() for x in want] + [1 << 20, 4 << 20]
        given = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in sizes]
        copies = [torch.empty_like(x) for x in given]
        torch.cuda.synchronize()
        torch.cuda._sleep(40_000_000)
        for x, y in zip(given, copies):
            y.copy_(x)
        del given, x
        got = call(side)
        side.synchronize()
        # bit for bit: the delta rule's state runs to NaN over these rows
        same = [torch.equal(*(t.cpu().view(torch.uint8) for t in pair)) for pair in zip((x for x in got if x is not None), want)]
        say(name, "NaN in", [int(x.isnan().sum()) for x in want if x.is_floating_point()])
        torch.cuda.synchronize()
        assert all(same), name
        assert all((y == 7).all() for y in copies), name
