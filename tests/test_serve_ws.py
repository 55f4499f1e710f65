"""CPU checks of the workspace of attention over a paged cache: what is asked for without a
window is enough for every window, so that a call with it is not refused for its
workspace.  Without a GPU such a call ends behind the checks, before anything is read."""
import ctypes
import random

import pytest

import tlgemm
from test_serve import P, attn


def no_gpu():
    import torch
    return not torch.cuda.is_available()


@pytest.mark.skipif(not no_gpu(), reason="the addresses are made up")
@pytest.mark.parametrize("type,kv", [(0, 0), (0, 1), (1, 1), (2, 2)])
def test_workspace_is_enough_for_every_window(type, kv):
    L, g = tlgemm.load(), random.Random(type * 3 + kv)
    for _ in range(8000):
        KV = g.choice([1, 2, 3, 8])
        H, hd, page = KV * g.choice([1, 2, 4, 5, 8]), g.choice([32, 64, 96, 128, 256]), g.choice([1, 16, 49, 64])
        B = g.choice([1, 2, 7, 40, 60, 300, 1100])
        N, ldt = int(B * 2 ** g.uniform(0, g.choice([3, 9]))), max(1, int(2 ** g.uniform(*g.choice([(3, 17), (9, 11)])) / page))
        c = dict(type=kv, KV=KV, hd=hd, page=page, page_ld=page * KV * hd, tok_ld=KV * hd, head_ld=hd)
        b = dict(B=B, N=N, ldt=ldt, max_rows=g.choice([0, 1, 6, N // B + 1, N]), max_len=g.choice([0, 100, ldt * page]))
        pages = tlgemm.pages(**{**dict(K=P, V=P, n_pages=8), **c})
        batch = tlgemm.batch(**{**dict(row0=P, len=P, table=P), **b})
        need = L.tlg_paged_attn_ws_bytes(ctypes.byref(pages), ctypes.byref(batch), type, H)
        for win, sinks in ((0, 0), (64, 4), (g.randint(300, 500), 0), (int(2 ** g.uniform(0, 17)), g.choice([0, 5, 600]))):
            rc = attn(L, c, b, type=type, ldq=H * hd, H=H, win=win, sinks=sinks, out=1 << 44, ldo=H * hd, ws_bytes=need)
            assert rc != 0 and "workspace" not in L.tlg_last_error().decode(), (c, b, H, win, sinks, L.tlg_last_error())
