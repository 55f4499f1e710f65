"""CPU checks of the serving operators (include/tlserve.h): every call that the
documentation rules out is refused before anything touches a GPU, and the
workspace sizes behave."""
import ctypes

import pytest

import tlgemm

EINVAL = -1
F32, F16, BF16 = tlgemm.F32, tlgemm.F16, tlgemm.BF16
P = 0x100000                            # an address that no refused call reads


@pytest.fixture(scope="module")
def L():
    return tlgemm.load()


def refused(L, rc, word):
    assert rc == EINVAL
    assert word in L.tlg_last_error().decode()


def args(c, b):
    pages = tlgemm.pages(**{**dict(K=P, V=P, type=F16, KV=2, hd=64, page=16, n_pages=8), **c})
    batch = tlgemm.batch(**{**dict(B=2, N=3, row0=P, len=P, table=P, ldt=4), **b})
    return ctypes.byref(pages), ctypes.byref(batch)


def store(L, c={}, b={}, q=P, ldq=256, q_out=P, ldqo=256, H=4, k=P, ldk=128, v=P, ldv=128, type=F16, cos=P, sin=P,
          maxpos=64):
    return L.tlg_dev_paged_store(*args(c, b), q, ldq, q_out, ldqo, H, k, ldk, v, ldv, type, cos, sin, maxpos, None)


def attn(L, c={}, b={}, q=P, type=F16, ldq=256, H=4, scale=0.1, win=0, sinks=0, out=2 * P, ldo=256, lse=P, ws=P,
         ws_bytes=1 << 40):
    return L.tlg_dev_paged_attn(*args(c, b), q, type, ldq, H, scale, win, sinks, out, ldo, lse, ws, ws_bytes, None)


def verify(L, x=P, type=F16, ld=8, scale=1.0, y=P, ldd=8, dscale=1.0, N=3, V=8, row0=P, B=2, draft=P, u=P, noise=P,
           ldn=8, tokens=P, logp=P, accepted=P, ws=P, ws_bytes=1 << 40):
    return L.tlg_dev_spec_verify(x, type, ld, scale, y, ldd, dscale, N, V, row0, B, draft, u, noise, ldn, tokens, logp,
                                 accepted, ws, ws_bytes, None)


BAD_BATCH = [dict(c=dict(type=3)), dict(c=dict(type=-1)), dict(type=3), dict(type=BF16), dict(c=dict(type=F32)),
             dict(c=dict(hd=48)), dict(c=dict(hd=0)), dict(c=dict(hd=512)), dict(c=dict(KV=0)), dict(c=dict(KV=1025)),
             dict(c=dict(page=0)), dict(c=dict(page=(1 << 16) + 1)), dict(c=dict(n_pages=-1)), dict(c=dict(K=None)),
             dict(c=dict(V=P + 8)), dict(c=dict(K=P + 2)), dict(c=dict(page_ld=2052)), dict(c=dict(tok_ld=132)),
             dict(c=dict(head_ld=-64)), dict(c=dict(head_ld=60)), dict(c=dict(page_ld=1 << 41)),
             dict(b=dict(B=-1)), dict(b=dict(B=(1 << 16) + 1)), dict(b=dict(N=-1)), dict(b=dict(N=(1 << 21) + 1)),
             dict(b=dict(ldt=-1)), dict(b=dict(ldt=1 << 27)), dict(b=dict(row0=None)), dict(b=dict(len=None)),
             dict(b=dict(table=None)), dict(b=dict(row0=P + 1)), dict(b=dict(max_rows=-1)), dict(b=dict(max_len=-1))]


@pytest.mark.parametrize("call,name", [(store, "paged_store"), (attn, "paged_attn")])
@pytest.mark.parametrize("bad", BAD_BATCH)
def test_bad_batches_are_refused(L, call, name, bad):
    refused(L, call(L, **bad), name)


@pytest.mark.parametrize("call", [store, attn])
def test_no_cache_or_batch_is_refused(L, call):
    c, b = args({}, {})
    for a in ((None, b), (c, None)):
        if call is store:
            rc = L.tlg_dev_paged_store(*a, None, 0, None, 0, 0, P, 128, P, 128, F16, None, None, 0, None)
        else:
            rc = L.tlg_dev_paged_attn(*a, P, F16, 256, 4, 0.1, 0, 0, P, 256, None, None, 0, None)
        assert rc == EINVAL


@pytest.mark.parametrize("bad", [dict(H=0), dict(H=1025), dict(q=P + 8), dict(ldq=255), dict(ldq=248), dict(ldq=260),
                                 dict(q_out=None), dict(ldqo=128), dict(k=None), dict(ldk=120), dict(ldk=132),
                                 dict(v=P + 4), dict(ldv=64), dict(cos=None), dict(sin=None), dict(cos=P + 4),
                                 dict(sin=P + 8), dict(maxpos=-1), dict(ldk=1 << 41), dict(ldqo=264), dict(q_out=P + 16),
                                 dict(q_out=P - 1024)])
def test_bad_stores_are_refused(L, bad):
    refused(L, store(L, **bad), "paged_store")


@pytest.mark.parametrize("bad", [dict(H=0), dict(H=3), dict(H=1026), dict(scale=0.0), dict(scale=-1.0),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-31),
                                 dict(scale=1e31), dict(win=-1), dict(sinks=-1), dict(q=None), dict(q=P + 8),
                                 dict(ldq=248), dict(ldq=260), dict(out=None), dict(out=P + 2), dict(ldo=128),
                                 dict(lse=P + 2), dict(out=P), dict(out=P + 1024), dict(out=P - 1520), dict(b=dict(N=1 << 20), H=514, ldq=514 * 64, ldo=514 * 64),
                                 dict(b=dict(B=1 << 16), c=dict(KV=65), H=65, ldq=65 * 64, ldo=65 * 64)])
def test_bad_attention_is_refused(L, bad):
    refused(L, attn(L, **bad), "paged_attn")


@pytest.mark.parametrize("bad", [dict(type=3), dict(N=-1), dict(N=(1 << 21) + 1), dict(V=0), dict(V=(1 << 20) + 1, ld=1 << 21),
                                 dict(ld=7), dict(x=None), dict(x=P + 1), dict(ldd=7), dict(y=P + 1),
                                 dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e31), dict(dscale=0.0),
                                 dict(dscale=1e-31), dict(B=-1), dict(B=(1 << 16) + 1), dict(row0=None),
                                 dict(row0=P + 2), dict(draft=None), dict(u=None), dict(noise=None), dict(tokens=None),
                                 dict(ldn=7), dict(noise=P + 1), dict(logp=P + 2), dict(accepted=P + 1), dict(ws=None),
                                 dict(ws=P + 8), dict(ws_bytes=0)])
def test_bad_verifications_are_refused(L, bad):
    refused(L, verify(L, **bad), "spec_verify")


def test_no_rows_is_no_work(L):
    """Calls without rows or sequences are valid and need no buffer and no GPU."""
    for b in (dict(N=0, row0=None, len=None, table=None), dict(B=0, row0=None, len=None, table=None)):
        assert store(L, b=b, q=None, k=None, v=None, cos=None, sin=None) == 0
        assert attn(L, b=b, q=None, out=None, lse=None, ws=None, ws_bytes=0) == 0
    assert verify(L, N=0, x=None, y=None, accepted=None, ws=None, ws_bytes=0) == 0
    assert verify(L, B=0, row0=None, ws=None, ws_bytes=0) == 0


@pytest.mark.parametrize("type", [F32, F16, BF16])
def test_verify_workspace(L, type):
    """A smaller, missing or unaligned workspace is refused, and none is large."""
    for N, V, B, d in ((1, 131072, 1, 1), (5, 2048, 2, 0), (300, 131072, 60, 1), (1, 1, 1, 1)):
        need = L.tlg_spec_verify_ws_bytes(type, N, V, B, d)
        assert need > 0
        for bad in (dict(ws_bytes=need - 1), dict(ws_bytes=need, ws=None), dict(ws_bytes=need, ws=P + 8)):
            refused(L, verify(L, type=type, N=N, V=V, B=B, ld=V, ldd=V, ldn=V, y=P if d else None, **bad),
                    "spec_verify: workspace")
    for N in (1, 7, 64, 5000, 1 << 21):
        for V in (1, 100, 50021, 1 << 20):
            for B in (1, 9, 1 << 16):
                assert 0 < L.tlg_spec_verify_ws_bytes(type, N, V, B, 1) <= 64 << 20


@pytest.mark.parametrize("type,kv", [(F32, F32), (F32, F16), (F16, F16), (BF16, BF16)])
def test_attention_workspace(L, type, kv):
    """What a call asks for is checked, and stays within bounds over all shapes."""
    for B, N, ldt, H, rows in ((1, 1, 8192, 32, 1), (1, 4096, 1024, 32, 4096), (64, 64, 256, 8, 1), (3, 30, 500, 4, 0),
                               (1, 1 << 21, 1 << 14, 4, 0), (1 << 16, 1 << 16, 100, 64, 1)):
        for hd in (32, 128, 256):
            c, b = args(dict(type=kv, hd=hd, KV=4), dict(B=B, N=N, ldt=ldt, max_rows=rows))
            need = L.tlg_paged_attn_ws_bytes(c, b, type, H)
            assert 0 <= need <= 256 << 20
            if need:
                for bad in (dict(ws_bytes=need - 1), dict(ws_bytes=need, ws=None), dict(ws_bytes=need, ws=P + 8)):
                    refused(L, attn(L, c=dict(type=kv, hd=hd, KV=4), b=dict(B=B, N=N, ldt=ldt, max_rows=rows), type=type,
                                    H=H, ldq=H * hd, ldo=H * hd, **bad), "paged_attn: workspace")
