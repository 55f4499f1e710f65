"""Scoring a text with the decoder (tl_decode_score) and distilling in the
training step (tl_train_set_teacher), alone and as a chain: a teacher's scores
become a student's targets."""
import math

import numpy as np
import pytest

from oracle import StepFns, model

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
KW = dict(V=128, D=96, L=3, H=3, KV=1, F=64, T=64)


@pytest.fixture(scope="module")
def host(lib):
    import tlgemm
    return tlgemm.host()


@pytest.fixture(scope="module")
def stream(lib):
    return lib.tlg_stream_create()


def weights(kw, seed):
    m = model(**kw)
    P = StepFns("oracle").init_params(m, seed)
    r = np.random.default_rng(seed)
    return P + (0.05 * r.standard_normal(P.size)).astype(np.float32)


def log_softmax(z):
    z = z - z.max(1, keepdims=True)
    return z - np.log(np.exp(z).sum(1, keepdims=True))


# (text length, W, mmax): one token, short of the bulk pass, into and past the
# ring, pieces of more than one bulk pass, odd chunks
CUTS = [(1, 64, 8), (7, 64, 8), (15, 64, 8), (16, 64, 8), (64, 64, 8), (65, 64, 8), (150, 64, 8), (40, 64, 3), (200, 100, 7),
        (30, 12, 4), (1100, 1100, 8)]


@pytest.mark.parametrize("opt", [dict(), dict(win=20, full_every=2, qknorm=1), dict(n_exp=2)], ids=str)
@pytest.mark.parametrize("cut", CUTS, ids=str)
def test_score(host, stream, cut, opt):
    """Against the log softmax, in 64 bits, of the logits that the same decoder
    leaves when it is fed chunk by chunk."""
    n, W, mmax = cut
    kw = dict(KW, **opt)
    r = np.random.default_rng(n)
    P = weights(kw, 3)
    tok = r.integers(0, KW["V"], n).astype(np.int32)
    K, temp = 9, 0.8
    a, b = (host.decode(kw, W, kv_f16=0, exact_exp=1, maxpos=2048, mmax=mmax, pool=1) for _ in range(2))
    a.upload(P, stream)
    b.upload(P, stream)
    lp, en, ti, tl = a.score(tok, stream, K=K, temp=temp)
    z = np.concatenate([b.chunk(tok[i:i + mmax], i, stream) for i in range(0, n, mmax)]).astype(np.float64)
    # the passes' logits agree to 1e-5 of their mean (sums in another order, as
    # prefill's are held to); a log probability moves by twice that / temp, and
    # carries the operator's own roundings
    dz = 1e-5 * np.abs(z).mean()
    ref = log_softmax(z / temp)
    tol = 2 * dz / temp + EPS * (4 * np.abs(ref).max() + 400)
    want = np.append(ref[np.arange(n - 1), tok[1:]], 0.0)
    assert lp[-1] == 0.0 and np.abs(lp - want).max() <= tol
    H = -(np.exp(ref) * ref).sum(1)
    assert np.abs(en - H).max() <= 2 * tol * (1 + np.log(KW["V"]))
    assert all(len(set(row)) == K for row in ti)
    best = -np.sort(-ref, axis=1)[:, :K]
    assert np.abs(np.take_along_axis(ref, ti.astype(np.int64), 1) - best).max() <= 2 * tol      # up to near ties
    assert np.abs(tl - best).max() <= tol
    assert (np.diff(tl, axis=1) <= 0).all()
    # the ring then holds the text: the next token decodes as after the chunks
    if n < 2048:
        x, y = (d.chunk(tok[:1], n, stream) for d in (a, b))
        assert np.abs(x - y).max() <= 1e-5 * np.abs(y).mean()
    # unfused, and without alternatives or entropy: the same call
    a.set_fused(0)
    lp2, _, _, _ = a.score(tok, stream, temp=temp)
    assert np.abs(lp2 - lp).max() <= 2 * tol


@pytest.mark.parametrize("opt", [dict(), dict(n_exp=2), dict(unfused=1)], ids=str)
@pytest.mark.parametrize("n", [1, 7, 16, 40, 64, 90])
def test_score_leaves_the_greedy_state(host, stream, n, opt):
    """Greedy decoding goes on after a score of the same text as if there had been
    none, eagerly and from a step captured before it: the next position and
    the token chosen for it are kept."""
    opt = dict(opt)
    unfused = opt.pop("unfused", 0)
    kw = dict(KW, **opt)
    tok = np.random.default_rng(n).integers(0, KW["V"], n).astype(np.int32)
    a, b = (host.decode(kw, 64, kv_f16=0, exact_exp=1, maxpos=256, mmax=8, pool=1) for _ in range(2))
    for d in (a, b):
        if unfused:
            d.set_fused(0)
        d.upload(weights(kw, 3), stream)
        d.prime(tok, stream)
    b.graph_build(stream)
    before = list(a.state(stream))
    assert list(b.state(stream)) == before
    for d in (a, b):
        d.score(tok, stream, K=3)
        assert list(d.state(stream)) == before
    want = host.decode(kw, 64, kv_f16=0, exact_exp=1, maxpos=256, mmax=8, pool=1)
    if unfused:
        want.set_fused(0)
    want.upload(weights(kw, 3), stream)
    want.prime(tok, stream)
    for _ in range(3):
        a.greedy_step(stream)
        b.graph_step(stream)
        want.greedy_step(stream)
        z = want.logits(1, stream)
        for d in (a, b):
            assert list(d.state(stream)) == list(want.state(stream))
            # the ring holds the same text, by passes whose sums differ in their order
            assert np.abs(d.logits(1, stream) - z).max() <= 1e-5 * np.abs(z).mean()


def test_score_refuses(host, stream):
    import tlgemm
    d = host.decode(KW, 64, maxpos=128)
    d.upload(weights(KW, 1), stream)
    ok = np.zeros(4, np.int32)
    for tok, K, temp in ((np.array([0, 128]), 0, 1.0), (np.array([-1]), 0, 1.0), (np.zeros(129), 0, 1.0), (ok, 129, 1.0),
                         (ok, -1, 1.0), (ok, 2, 0.0), (ok, 2, math.nan)):
        with pytest.raises((tlgemm.TlgError, ValueError)):
            d.score(tok, stream, K=K, temp=temp)
    d.score(ok, stream, K=2)


def train_state(host, lib, stream, B=3, kw=KW):
    tr = host.train(kw, B)
    r = np.random.default_rng(5)
    tok, tgt = (r.integers(0, kw["V"], tr.N).astype(np.int32) for _ in range(2))
    P = weights(kw, 7)

    def start():
        tr.upload(P, stream)
        tr.set_batch(tok, tgt, None, stream)
        tr.set_hyper(1e-3, 0.9, 0.95, 0.1, 1, stream)
    start()
    return tr, tok, tgt, start


def buf(lib, ptr, shape, stream):
    a = np.empty(shape, np.float32)
    lib.check(lib.tlg_memcpy_d2h(a.ctypes.data, ptr, a.nbytes, stream), "d2h")
    lib.check(lib.tlg_stream_sync(stream), "sync")
    return a


def reference(z, ids, logp, tail, temp, w_kd, tgt, w_ce):
    """Rows and d rows / d logits in 64 bits."""
    N, V = z.shape
    lp, lp1 = log_softmax(z / temp), log_softmax(z)
    rows, grad = np.zeros(N), np.zeros((N, V))
    for n in range(N):
        on = ids[n] >= 0
        q = np.zeros(V)
        q[ids[n][on]] = np.exp(logp[n][on].astype(np.float64))
        inside = np.zeros(V, bool)
        inside[ids[n][on]] = True
        qr = max(0.0, 1.0 - q.sum()) if tail and on.any() else 0.0
        if not tail and on.any():
            q /= q.sum()
        p = np.exp(lp[n])
        s = q > 0
        rows[n] = (q[s] * (np.log(q[s]) - lp[n][s])).sum()
        mass = np.full(V, q.sum() + qr)
        if qr > 0:
            pr = p[~inside].sum()
            rows[n] += qr * (math.log(qr) - math.log(pr))
            mass[~inside] -= qr / pr
        rows[n] = w_kd * temp * temp * rows[n] - w_ce * lp1[n, tgt[n]]
        grad[n] = w_kd * temp * (mass * p - q) + w_ce * np.exp(lp1[n])
        grad[n, tgt[n]] -= w_ce
    return rows, grad


@pytest.mark.parametrize("tail,temp,w_ce", [(False, 2.0, 0.4), (True, 1.0, 0.0)])
def test_a_teacher_scores_and_a_student_learns(host, lib, stream, tail, temp, w_ce):
    """Teacher: the decoder scores every sequence of the batch.  Student: the
    training step's loss and head gradient are the distillation's of its own
    logits, and captured steps equal eager ones bit for bit."""
    B, K, V = 3, 12, KW["V"]
    tr, tok, tgt, start = train_state(host, lib, stream, B)
    teacher = host.decode(KW, KW["T"], kv_f16=0, exact_exp=1, maxpos=256)
    teacher.upload(weights(KW, 11), stream)
    got = [teacher.score(s, stream, K=K, temp=temp) for s in tok.reshape(B, -1)]
    ids, logp = np.concatenate([g[2] for g in got]), np.concatenate([g[3] for g in got])
    ids[KW["T"] - 1] = -1                                # a row without a teacher
    tr.set_teacher(ids, logp, stream, tail=tail, temp=temp, w_kd=0.6, w_ce=w_ce)
    tr.forward(stream)
    z = buf(lib, tr.act("logits"), (tr.N, V), stream).astype(np.float64)
    rows, grad = reference(z, ids, logp, tail, temp, 0.6, tgt, w_ce)
    d = buf(lib, tr.act("dlogits"), (tr.N, V), stream)
    # log probabilities of 128 tokens: |z' - log S| <= 20, sums of 128 terms
    tol = (0.6 * temp * temp * 3 + w_ce) * EPS * (4 * 20 + 150)
    assert abs(tr.loss(stream) - rows.mean()) <= tol + 2 * EPS * abs(rows.mean())
    assert np.abs(d - grad / tr.N).max() <= (tol * 3 + 4 * EPS) / tr.N
    tr.backward(stream)

    def run(step):
        start()
        out = []
        for it in range(3):
            tr.set_hyper(1e-3, 0.9, 0.95, 0.1, it + 1, stream)
            step(stream)
            out.append((tr.loss(stream), tr.gnorm(stream)))
        return out, buf(lib, tr.buf(0), tr.np, stream)
    eager = run(tr.step)
    tr.graph_build(stream)
    for _ in range(2):
        replay = run(tr.graph_step)
        assert eager[0] == replay[0] and np.array_equal(eager[1], replay[1])
    # new contents of the same shape: the captured step takes them
    tr.set_teacher(np.roll(ids, 1, 0), np.roll(logp, 1, 0), stream, tail=tail, temp=temp, w_kd=0.6, w_ce=w_ce)
    second = run(tr.graph_step)
    assert second[0] != eager[0]
    assert second[0] == run(tr.step)[0]


def test_without_a_teacher_the_step_is_as_before(host, lib, stream):
    """Going back to the cross-entropy gives the same bits as never having left
    it, and a captured step of the other loss is not replayed."""
    import tlgemm
    tr, tok, tgt, start = train_state(host, lib, stream)
    tr.step(stream)
    before = tr.loss(stream), buf(lib, tr.buf(0), tr.np, stream)
    tr.graph_build(stream)
    ids = np.tile(np.arange(4, dtype=np.int32), (tr.N, 1))
    tr.set_teacher(ids, np.full(ids.shape, -2.0), stream, w_kd=1.0, w_ce=0.5)
    with pytest.raises(tlgemm.TlgError):
        tr.graph_step(stream)
    start()
    tr.step(stream)
    assert tr.loss(stream) != before[0]
    tr.graph_build(stream)
    tr.set_teacher(None, None, stream)
    with pytest.raises(tlgemm.TlgError):
        tr.graph_step(stream)
    start()
    tr.step(stream)
    assert tr.loss(stream) == before[0] and np.array_equal(buf(lib, tr.buf(0), tr.np, stream), before[1])


def test_set_teacher_refuses(host, lib, stream):
    import tlgemm
    tr, tok, tgt, start = train_state(host, lib, stream)
    ids, lp = np.zeros((tr.N, 3), np.int32), np.full((tr.N, 3), -1.0)
    bad = ids.copy()
    bad[5, 1] = KW["V"]
    for i, l, kw in ((bad, lp, {}), (ids, lp, dict(temp=0.0)), (ids, lp, dict(temp=math.nan)), (ids, lp, dict(w_kd=math.inf)),
                     (ids, lp, dict(w_ce=math.nan)), (np.zeros((tr.N, 129), np.int32), np.zeros((tr.N, 129)), {})):
        with pytest.raises(tlgemm.TlgError):
            tr.set_teacher(i, l, stream, **kw)
    tr.set_teacher(ids, lp, stream, w_ce=1.0)
    tr.step(stream)
    assert math.isfinite(tr.loss(stream))


def test_broken_teachers_are_refused(host, lib, stream):
    """Log probabilities of NaN or +inf never train: set_teacher refuses them at
    entries, and rows as a decoder with NaN weights scores them; the teacher that
    was there stays.  Padding may hold anything else."""
    import tlgemm
    tr, tok, tgt, start = train_state(host, lib, stream)
    ids, lp = np.zeros((tr.N, 3), np.int32), np.full((tr.N, 3), -1.5)
    ids[:, 1], ids[:, 2] = 1, 2
    tr.set_teacher(ids, lp, stream)
    tr.step(stream)
    loss = tr.loss(stream)
    for v in (math.nan, math.inf):
        bad = lp.copy()
        bad[7, 2] = v
        with pytest.raises(tlgemm.TlgError):
            tr.set_teacher(ids, bad, stream)
    P = weights(KW, 11)
    P[5 * KW["D"]] = math.nan                            # token 5's embedding: every row's logits
    broken = host.decode(KW, KW["T"], kv_f16=0, exact_exp=1, maxpos=256)
    broken.upload(P, stream)
    got = [broken.score(s, stream, K=3) for s in tok.reshape(-1, KW["T"])]
    bids, blp = np.concatenate([g[2] for g in got]), np.concatenate([g[3] for g in got])
    assert (bids == -1).all() and np.isnan(blp).all()
    with pytest.raises(tlgemm.TlgError):
        tr.set_teacher(bids, blp, stream)
    one = np.where(np.arange(tr.N)[:, None] == 3, bids, ids), np.where(np.arange(tr.N)[:, None] == 3, blp, lp)
    with pytest.raises(tlgemm.TlgError):
        tr.set_teacher(one[0], one[1], stream)
    start()
    tr.step(stream)
    assert tr.loss(stream) == loss
    ids[3], lp[3, 0], lp[3, 1:] = -1, -math.inf, math.nan                # padding
    ids[4, 2], lp[4, 2] = -1, math.nan
    tr.set_teacher(ids, lp, stream)
    start()
    tr.step(stream)
    assert math.isfinite(tr.loss(stream))
