"""CPU checks of the vocabulary operators (include/tltrain.h): every call that
the documentation rules out is refused before anything touches a GPU, and the
workspace sizes behave."""
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


def lp(L, logits=P, type=F32, ld=8, N=2, V=8, scale=1.0, ids=P, M=1, logp=P, lse2=P, entropy=P, K=2, top_ids=P,
       top_logp=P, ws=P, ws_bytes=1 << 30):
    return L.tlg_dev_logprobs(logits, type, ld, N, V, scale, ids, M, logp, lse2, entropy, K, top_ids, top_logp, ws,
                              ws_bytes, None)


def bwd(L, logits=P, type=F32, ld=8, N=2, V=8, scale=1.0, ids=P, M=1, lse2=P, entropy=P, dlogp=P, dlse=None,
        dent=None, d=2 * P, ldd=8):
    return L.tlg_dev_logprobs_bwd(logits, type, ld, N, V, scale, ids, M, lse2, entropy, dlogp, dlse, dent, d, ldd,
                                  None)


def kd(L, logits=P, type=F32, ld=8, N=2, V=8, t_ids=P, t_logp=P, K=2, tail=0, temp=1.0, w_kd=1.0, tgt=P, w_ce=0.5,
       rows=P, loss=P, d=2 * P, ldd=8, scale=1.0, ws=P, ws_bytes=1 << 30):
    return L.tlg_dev_distill(logits, type, ld, N, V, t_ids, t_logp, K, tail, temp, w_kd, tgt, w_ce, rows, loss, d,
                             ldd, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("call,name", [(lp, "logprobs"), (bwd, "logprobs_bwd"), (kd, "distill")])
@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(N=-1), dict(N=(1 << 21) + 1), dict(V=0), dict(V=-5), dict(ld=7),
                                 dict(V=(1 << 20) + 1, ld=1 << 21), dict(logits=None), dict(logits=P + 2),
                                 dict(type=F16, logits=P + 1), dict(type=BF16, logits=P + 1)])
def test_bad_rows_are_refused(L, call, name, bad):
    refused(L, call(L, **bad), name)


@pytest.mark.parametrize("bad", [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(scale=1e-31), dict(scale=1e31), dict(M=-1), dict(M=65), dict(K=-1), dict(K=129),
                                 dict(ids=None), dict(logp=None), dict(top_ids=None), dict(top_logp=None)])
def test_bad_logprobs_are_refused(L, bad):
    refused(L, lp(L, **bad), "logprobs")


@pytest.mark.parametrize("bad", [dict(scale=0.0), dict(scale=float("nan")), dict(M=65), dict(ids=None),
                                 dict(dlogp=None), dict(lse2=None), dict(entropy=None, dent=P), dict(d=None),
                                 dict(ldd=7), dict(d=2 * P + 1), dict(d=P + 4), dict(d=P, ldd=9), dict(d=P - 32)])
def test_bad_gradients_are_refused(L, bad):
    refused(L, bwd(L, **bad), "logprobs_bwd")


@pytest.mark.parametrize("bad", [dict(temp=0.0), dict(temp=-2.0), dict(temp=1e-38), dict(temp=1e38), dict(temp=float("nan")), dict(w_kd=float("inf")),
                                 dict(w_ce=float("nan")), dict(scale=float("nan")), dict(K=-1), dict(K=129),
                                 dict(t_ids=None), dict(t_logp=None), dict(tgt=None), dict(rows=None, loss=P),
                                 dict(rows=None, loss=None, d=None), dict(ldd=7), dict(d=P + 4), dict(d=P, ldd=9)])
def test_bad_distillations_are_refused(L, bad):
    refused(L, kd(L, **bad), "distill")


def test_no_rows_is_no_work(L):
    """N = 0 is a valid call that needs no buffer and no GPU."""
    assert lp(L, N=0, logits=None, ids=None, logp=None, top_ids=None, top_logp=None, ws=None, ws_bytes=0) == 0
    assert bwd(L, N=0, logits=None, ids=None, lse2=None, dlogp=None, d=None) == 0
    assert kd(L, N=0, logits=None, t_ids=None, t_logp=None, tgt=None, rows=None, loss=None, d=None, ws=None,
              ws_bytes=0) == 0


@pytest.mark.parametrize("type", [F32, F16, BF16])
def test_workspace_is_needed_and_checked(L, type):
    """Few rows of a large vocabulary are cut over workgroups and need a
    workspace; a batch that fills the chip needs none.  A smaller or missing
    one is refused."""
    V = 131072
    need = L.tlg_logprobs_ws_bytes(type, 1, V, 20)
    assert need == 0 or lp(L, type=type, N=1, V=V, ld=V, K=20, ws_bytes=need - 1) == EINVAL
    assert need == 0 or lp(L, type=type, N=1, V=V, ld=V, K=20, ws=None, ws_bytes=need) == EINVAL
    assert need == 0 or lp(L, type=type, N=1, V=V, ld=V, K=20, ws=P + 8, ws_bytes=need) == EINVAL
    need = L.tlg_distill_ws_bytes(type, 1, V)
    assert need == 0 or kd(L, type=type, N=1, V=V, ld=V, ldd=V, d=1 << 40, ws_bytes=need - 1) == EINVAL
    assert need == 0 or kd(L, type=type, N=1, V=V, ld=V, ldd=V, d=1 << 40, ws=None, ws_bytes=need) == EINVAL
    assert L.tlg_logprobs_ws_bytes(type, 4096, 2048, 32) == 0
    assert L.tlg_distill_ws_bytes(type, 4096, 2048) == 0
    # never more than a few MiB, whatever the rows
    for N in (1, 2, 7, 64, 500, 4096, 1 << 20):
        for V in (1, 100, 2048, 50021, 131072, 1 << 20):
            assert 0 <= L.tlg_logprobs_ws_bytes(type, N, V, 128) <= 16 << 20
            assert 0 <= L.tlg_distill_ws_bytes(type, N, V) <= 16 << 20


@pytest.mark.parametrize("ids,logp", [((5, 3), (4, 3)), ((5, 3), (4, 2)), ((4, 3), (4, 4)), ((4,), (4,)), ((3, 3), (3, 3))])
def test_teachers_of_another_shape_are_refused(ids, logp):
    """Before the arrays reach the library, with or without assertions (-O)."""
    from types import SimpleNamespace as NS

    import numpy as np
    tr = object.__new__(tlgemm.Train)
    tr.N, tr.h = 4, None

    def call(*args):
        raise RuntimeError("read past an array")
    tr.host = NS(dll=NS(tl_train_set_teacher=call))
    with pytest.raises(ValueError):
        tr.set_teacher(np.zeros(ids, np.int32), np.zeros(logp, np.float32), None)


@pytest.mark.parametrize("type", [F32, F16, BF16])
def test_cut_rows_need_their_workspace(L, type):
    """One row of 131072 columns is cut for every type and both operators, and
    refused without the workspace or with a smaller or unaligned one."""
    V = 131072
    need = L.tlg_logprobs_ws_bytes(type, 1, V, 20)
    assert need > 0 and L.tlg_distill_ws_bytes(type, 1, V) > 0
    for bad in (dict(ws_bytes=need - 1), dict(ws_bytes=need, ws=None), dict(ws_bytes=need, ws=P + 8)):
        refused(L, lp(L, type=type, N=1, V=V, ld=V, K=20, **bad), "logprobs: workspace")
    need = L.tlg_distill_ws_bytes(type, 1, V)
    for bad in (dict(ws_bytes=need - 1), dict(ws_bytes=need, ws=None), dict(ws_bytes=need, ws=P + 8)):
        refused(L, kd(L, type=type, N=1, V=V, ld=V, ldd=V, d=1 << 40, **bad), "distill: workspace")
