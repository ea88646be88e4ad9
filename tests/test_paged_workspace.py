"""What lmxp_attn_workspace_bytes promises, on the CPU (calls return before anything is
enqueued)."""
import ctypes
import random

import pytest

import llmoxide_amd as lmx
from llmoxide_amd import paged
from tests.test_paged import FAKE, FAR, S, attn, batch, pool


def workspace(p, b, heads, window=0):
    d = paged.PagedAttnDesc(n_heads=heads, window=window, q_head_stride=0, q_row_stride=0, scale=0.1)
    return paged.paged_lib().lmxp_attn_workspace_bytes(ctypes.byref(p), ctypes.byref(b), ctypes.byref(d))


def wide(kv=8, hd=128, page=16, store=paged.STORE_F16):
    scales = dict(k_scale=FAKE, v_scale=FAKE) if store == paged.STORE_I8 else {}
    return pool(n_pages=1 << 20, n_kv_heads=kv, head_dim=hd, page_size=page, store=store, **scales)


def rows(seqs, tokens, new, ctx):
    return batch(n_seq=seqs, n_tokens=tokens, max_new=new, max_ctx=ctx, table_stride=1 << 20)


SHAPES = [(8, 4, 128), (8, 1, 64), (1, 1, 128), (2, 8, 256), (4, 5, 512), (1, 16, 512), (300, 1, 128)]


@pytest.mark.parametrize("kv,group,hd", SHAPES)
@pytest.mark.parametrize("store", [paged.STORE_F16, paged.STORE_I8])
def test_the_workspace_of_a_batch_serves_every_smaller_one(kv, group, hd, store):
    rng = random.Random(kv * hd + store)
    p = wide(kv=kv, hd=hd, store=store)

    def most(hi):
        return max(1, min(hi, int(2 ** rng.uniform(0, 14))))
    for _ in range(400):
        tokens = most(1 << 14)
        big = (most(40), tokens, most(tokens), most(1 << 14))
        tokens = most(tokens)
        small = (most(big[0]), tokens, most(min(tokens, big[2])), most(big[3]))
        window = rng.choice([0, 1, 100, 1 << 20])
        need, has = workspace(p, rows(*small), kv * group, window), workspace(p, rows(*big), kv * group)
        assert need <= has, (small, big, window)


@pytest.mark.parametrize("seqs,ctx,small", [
    (1, 32768, (1, 512, 512)), (1, 32768, (1, 1, 1)), (1, 8192, (1, 300, 300)), (33, 8192, (33, 544, 512)),
    (33, 8192, (4, 4, 1)),
])
@pytest.mark.parametrize("dt", [lmx.F32, lmx.F16])
@pytest.mark.parametrize("window", [0, 4000])
def test_calls_take_the_workspace_of_a_larger_batch(seqs, ctx, small, dt, window):
    """Each small batch is cut between workgroups, in a window too: its call needs a workspace,
    and goes on past its size to the next check (the alignment), which refuses it."""
    p = wide()
    has = workspace(p, rows(seqs, 8192, 8192, ctx), 32)
    call = dict(p=p, b=rows(*small, ctx), dt=dt, n_heads=32, window=window, out=FAR * 16, ws=FAKE + 8)
    assert attn(ws_bytes=0, **call) == S.E_WORKSPACE
    assert attn(ws_bytes=has, **call) == S.E_ALIGN


@pytest.mark.parametrize("window", [0, 2500, 2501, 1 << 20])
def test_a_window_that_hides_nothing_is_none(window):
    """2500 rows of 8 heads of 256 are split without a window, and so behind one as long as
    the sequence."""
    b = rows(1, 2500, 2500, 2500)
    call = dict(p=wide(hd=256), b=b, dt=lmx.F16, n_heads=8, out=FAR * 16, ws=FAKE + 8, window=window)
    assert attn(ws_bytes=0, **call) == S.E_WORKSPACE
    assert attn(ws_bytes=workspace(wide(hd=256), b, 8, window), **call) == S.E_ALIGN


def test_streams_and_workspaces_of_another_device_are_refused(monkeypatch):
    """Stand-ins for what two GPUs would give: the check reads nothing but devices."""
    torch = pytest.importorskip("torch")

    class On:
        def __init__(self, index):
            self.device = torch.device("cuda", index)
            self.device_index = index

        def get_device(self):
            return self.device.index

    class Space:
        def __init__(self, buf=None, device=None):
            self.buf, self.device = buf, device
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    here, there = On(0), On(1)
    paged._place(here, here, here, None, stream=here, workspace=Space(buf=here))
    for device in (None, "cuda", "cuda:0", torch.device("cuda"), 0):
        paged._place(here, here, workspace=Space(device=device))
    for kw in (dict(stream=there), dict(workspace=Space(buf=there)), dict(workspace=Space(buf=there, device="cuda:0")),
               dict(workspace=Space(device="cuda:1")), dict(workspace=Space(device=1))):
        with pytest.raises(ValueError):
            paged._place(here, here, here, **kw)
    for args in ((here, there), (there, there), (here, here, there)):
        with pytest.raises(ValueError):
            paged._place(*args)
