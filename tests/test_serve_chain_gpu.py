"""The serving operators as they are used: a batch of sequences through a whole
model over a paged cache, with drafts verified by sampling, against the decoder
of one sequence; and the decoder's own sampled self-speculative generation
(tl_decode_sample_spec)."""
import math

import numpy as np
import pytest

import tlgemm
from oracle import StepFns, model
from test_serve_gpu import F16, F32, ints, ref_verify

pytestmark = pytest.mark.gpu
KW = dict(V=128, D=128, L=2, H=4, KV=1, F=96, T=256)
HD, PAGE, MASK = 32, 16, (1 << 64) - 1


def _t():
    import torch
    return torch


def weights(kw, seed):
    m = model(**kw)
    P = StepFns("oracle").init_params(m, seed)
    return m, P + (0.08 * np.random.default_rng(seed).standard_normal(P.size)).astype(np.float32)


@pytest.fixture(scope="module")
def host(lib):
    return tlgemm.host()


@pytest.fixture(scope="module")
def stream(lib):
    return lib.tlg_stream_create()


class Server:
    """forward_chunk for a batch: every sequence's new tokens through the library's
    own entries, the attention over a paged cache.  Buffers have room for `rows`."""

    def __init__(self, lib, m, P, kv, pages, rows, maxpos=256):
        t = _t()
        self.lib, self.m, self.kv, self.rows = lib, m, kv, rows
        self.P = t.from_numpy(P).cuda()
        self.maps = [StepFns("oracle").layer_map(m, l) for l in range(m.L)]
        KD = m.KV * HD
        self.caches = [[t.full((pages, PAGE, KD), float("nan"), dtype=t.float16 if kv == F16 else t.float32, device="cuda")
                        for _ in range(2)] for _ in range(m.L)]
        ang = np.arange(maxpos)[:, None] * 10000.0 ** (-2.0 * np.arange(HD // 2) / HD)
        self.cos, self.sin = (t.from_numpy(f(ang).astype(np.float32)).cuda() for f in (np.cos, np.sin))
        self.maxpos = maxpos
        f = lambda *s: t.zeros(rows, *s, device="cuda")
        self.x, self.n, self.q, self.k, self.v = f(m.D), f(m.D), f(m.D), f(KD), f(KD)
        self.qr, self.ctx, self.y, self.act, self.logits = f(m.D), f(m.D), f(m.D), f(m.F), f(m.V)

    def w(self, l, name):
        return self.P.data_ptr() + 4 * self.maps[l][name]

    def forward(self, tokens, row0, lens, table, max_rows, max_len):
        """Logits [N][V] of the new tokens (device ints); row0, lens and table on the GPU."""
        L, m, N, st = self.lib, self.m, tokens.numel(), _t().cuda.current_stream().cuda_stream
        D, KD, F, V = m.D, m.KV * HD, m.F, m.V
        p = lambda z: z.data_ptr()
        batch = tlgemm.batch(lens.numel(), N, p(row0), p(lens), p(table), table.shape[1], max_rows, max_len)
        L.check(L.tlg_dev_embed_fwd(p(self.x), self.w(0, "emb"), p(tokens), N, D, V, st))
        for l in range(m.L):
            pages = tlgemm.pages(p(self.caches[l][0]), p(self.caches[l][1]), self.kv, m.KV, HD, PAGE,
                                 self.caches[l][0].shape[0])
            L.check(L.tlg_dev_rmsnorm_fwd(p(self.x), self.w(l, "an1"), p(self.n), None, N, D, st))
            L.group([dict(op="mm", C=p(c), M=N, K=D, N=w, A=[p(self.n)], B=[self.w(l, name)])
                     for c, w, name in ((self.q, D, "wq"), (self.k, KD, "wk"), (self.v, KD, "wv"))], st)
            L.paged_store(pages, batch, p(self.q), D, p(self.qr), D, m.H, p(self.k), KD, p(self.v), KD, F32, p(self.cos),
                          p(self.sin), self.maxpos, st)
            nb = L.paged_attn_ws_bytes(pages, batch, F32, m.H)
            ws = _t().empty(max(nb, 16), dtype=_t().uint8, device="cuda")
            L.paged_attn(pages, batch, p(self.qr), F32, D, m.H, HD ** -0.5, 0, 0, p(self.ctx), D, None, p(ws), nb, st)
            L.group([dict(op="mm", C=p(self.y), M=N, K=D, N=D, A=[p(self.ctx)], B=[self.w(l, "wo")])], st)
            L.check(L.tlg_dev_add(p(self.y), p(self.x), N * D, st))
            L.check(L.tlg_dev_rmsnorm_fwd(p(self.y), self.w(l, "an2"), p(self.n), None, N, D, st))
            L.check(L.tlg_dev_swiglu_mm(p(self.n), self.w(l, "w1"), self.w(l, "w3"), p(self.act), None, None, N, D, F, st))
            L.group([dict(op="mm", C=p(self.x), M=N, K=F, N=D, A=[p(self.act)], B=[self.w(l, "w2")])], st)
            L.check(L.tlg_dev_add(p(self.x), p(self.y), N * D, st))
        L.check(L.tlg_dev_rmsnorm_fwd(p(self.x), self.w(0, "nf"), p(self.n), None, N, D, st))
        L.group([dict(op="mm_bt", beta=0, C=p(self.logits), M=N, K=V, N=D, A=[p(self.n)], B=[self.w(0, "emb")])], st)
        return self.logits[:N]


@pytest.mark.parametrize("kv", [F32, F16])
def test_batch_over_pages(lib, host, stream, kv):
    """Three prompts of different lengths at once, then rounds of a token and two
    drafts each, some kept and some not: the logits of every row are those of a
    decoder that is fed the same sequence alone (its ring as large as the text),
    to the order of the sums, and what the verification keeps is what its
    definition says about these logits."""
    t = _t()
    m, P = weights(KW, 5)
    g = np.random.default_rng(6)
    prompts = [g.integers(0, m.V, n).astype(np.int32) for n in (20, 37, 5)]
    B, V = len(prompts), m.V
    srv = Server(lib, m, P, kv, pages=30, rows=80)
    # pages as sequences ask for them, in random order
    free, table = list(g.permutation(30)), np.full((B, 9), -1, np.int32)

    def room(b, n):
        for i in range(-(-n // PAGE)):
            if table[b, i] < 0:
                table[b, i] = free.pop()
    decs = []
    for pr in prompts:
        d = host.decode(KW, 256, kv_f16=int(kv == F16), exact_exp=1, maxpos=256, mmax=8)
        d.upload(P, stream)
        decs.append(d)
    texts, feeds, drafts_of = [list(p) for p in prompts], [list(p) for p in prompts], [0] * B
    for rnd in range(5):
        lens = [len(texts[b]) - 1 + len(feeds[b]) if rnd else len(feeds[b]) for b in range(B)]
        for b in range(B):
            room(b, lens[b])
        row0 = np.concatenate([[0], np.cumsum([len(f) for f in feeds])])
        flat = [x for f in feeds for x in f]
        z = srv.forward(ints(flat), ints(row0), ints(lens), t.from_numpy(table).cuda(), max(map(len, feeds)), max(lens))
        t.cuda.synchronize()
        logits = z.cpu().numpy().copy()
        for b in range(B):                    # the same rows by the decoder of one sequence
            start = lens[b] - len(feeds[b])
            want = np.concatenate([decs[b].chunk(np.array(feeds[b][i:i + 8], np.int32), start + i, stream)
                                   for i in range(0, len(feeds[b]), 8)])
            got = logits[row0[b]:row0[b + 1]]
            tol = (2e-5 if kv == F32 else 2e-3) * abs(want).max()        # fp16 keys round apart where sums differ
            assert abs(got - want).max() <= tol, (rnd, b, abs(got - want).max(), tol)
        # verification: in the first round only the prompts' last rows are sampled from
        first = [row0[b + 1] - 1 - drafts_of[b] for b in range(B)]
        pick = [r for b in range(B) for r in range(first[b], row0[b + 1])]
        vrow0 = np.concatenate([[0], np.cumsum([drafts_of[b] + 1 for b in range(B)])])
        draft = np.full(len(pick), -1, np.int32)
        for b in range(B):
            draft[vrow0[b]:vrow0[b + 1] - 1] = feeds[b][1:] if drafts_of[b] else []
        zz = t.from_numpy(logits[pick]).cuda()
        u, e = t.from_numpy(g.random(len(pick)).astype(np.float32)).cuda(), \
            t.from_numpy(g.exponential(size=(B, V)).astype(np.float32)).cuda()
        tok, acc = t.zeros(len(pick), dtype=t.int32, device="cuda"), t.zeros(B, dtype=t.int32, device="cuda")
        nb = lib.tlg_spec_verify_ws_bytes(F32, len(pick), V, B, 0)
        ws = t.empty(nb, dtype=t.uint8, device="cuda")
        dr, dd = ints(vrow0), ints(draft)
        lib.spec_verify(zz.data_ptr(), F32, V, 1.25, None, 0, 1.0, len(pick), V, dr.data_ptr(), B, dd.data_ptr(),
                        u.data_ptr(), e.data_ptr(), V, tok.data_ptr(), None, acc.data_ptr(), ws.data_ptr(), nb,
                        t.cuda.current_stream().cuda_stream)
        tok, acc = tok.cpu().numpy(), acc.cpu().numpy()
        want, _, wacc = ref_verify(logits[pick].astype(np.float64), None, vrow0, draft, u.cpu().double().numpy(),
                                   e.cpu().double().numpy(), 1.25, 1.0)
        assert (tok == want).all() and (acc == wacc).all()
        for b in range(B):
            texts[b] += [int(x) for x in tok[vrow0[b]:vrow0[b] + acc[b] + 1]]
            likely = np.argsort(-logits[pick][vrow0[b] + acc[b]])
            feeds[b] = [texts[b][-1], int(likely[0]), int(likely[1 + rnd % 2])]
            drafts_of[b] = 2
    assert len(free) < 30 - 3


def bits(seed, i):
    z = (seed + (i + 1) * 0x9E3779B97F4A7C15) & MASK
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & MASK
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & MASK
    return z ^ (z >> 31)


def numbers(seed, call, V):
    base = call * (V + 8)
    u = np.array([(bits(seed, base + r) >> 40) * 2.0 ** -24 for r in range(8)])
    e = np.array([-math.log(((bits(seed, base + 8 + v) >> 11) + 0.5) * 2.0 ** -53) for v in range(V)])
    return u, e.astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("n_mtp,mmax", [(3, 8), (1, 2), (0, 1), (3, 3)])
@pytest.mark.parametrize("temp", [1.0, 0.4])
def test_sample_spec(lib, host, stream, n_mtp, mmax, temp):
    """Round for round against the definition: the same chunks by hand through a
    second decoder, its heads' drafts, and a float64 verification of its logits
    with the documented numbers."""
    t = _t()
    kw = dict(KW, n_mtp=n_mtp)
    m, P = weights(kw, 7)
    prompt, n, seed = np.arange(3, 14, dtype=np.int32), 21, 12345678901234567
    a, b = (host.decode(kw, 64, kv_f16=0, exact_exp=1, maxpos=64, mmax=mmax) for _ in range(2))
    a.upload(P, stream)
    b.upload(P, stream)
    toks, lp, chunks = a.sample_spec(prompt, n, stream, temp=temp, seed=seed)
    again, lp2, c2 = a.sample_spec(prompt, n, stream, temp=temp, seed=seed)
    assert (again == toks).all() and (lp2 == lp).all() and c2 == chunks
    other, _, _ = a.sample_spec(prompt, n, stream, temp=temp, seed=seed + 1)
    assert (other != toks).any()

    V, heads = m.V, min(n_mtp, mmax - 1)
    for i in range(0, len(prompt), mmax):
        z = b.chunk(prompt[i:i + mmax], i, stream)
    cur, pos, call, want, wlp, dtok = len(z) - 1, len(prompt), 0, [], [], t.zeros(8, dtype=t.int32, device="cuda")
    t.cuda.synchronize()
    drafts, rows = [], z[cur:cur + 1]
    while True:
        u, e = numbers(seed, call, V)
        k = len(drafts)
        tk, tl, acc = ref_verify(rows.astype(np.float64), None, [0, k + 1], np.array(drafts + [-1]), u[:k + 1], e[None],
                                 1.0 / temp, 1.0)
        got = int(acc[0]) + 1
        want += [int(x) for x in tk[:got]]
        wlp += list(tl[:got])
        if call:
            cur, pos = int(acc[0]), pos + got
        call += 1
        if len(want) >= n:
            break
        drafts = []
        for h in range(min(heads, n - len(want) - 1, 64 - pos - 1)):
            b.mtp_draft(cur, h, dtok.data_ptr() + 4 * h, stream)
            lib.check(lib.tlg_stream_sync(stream))
            drafts.append(int(dtok[h]))
        rows = b.chunk(np.array([want[-1]] + drafts, np.int32), pos, stream)
    assert list(toks) == want and chunks == call - 1
    assert abs(lp - np.array(wlp)).max() <= 1e-5 * (1 + abs(np.array(wlp)).max())


def test_sample_spec_cold_is_greedy(lib, host, stream):
    """At a temperature towards 0 the samples are the greedy tokens."""
    kw = dict(KW, n_mtp=2)
    m, P = weights(kw, 8)
    prompt = np.arange(40, 49, dtype=np.int32)
    d = host.decode(kw, 128, kv_f16=1, exact_exp=0, maxpos=128, mmax=8)
    d.upload(P, stream)
    greedy, _ = d.generate_spec(prompt, 30, stream)
    got, lp, _ = d.sample_spec(prompt, 30, stream, temp=1e-6, seed=3)
    assert list(got) == list(greedy) and abs(lp).max() <= 1e-3


def test_sample_spec_refusals(lib, host, stream):
    m, P = weights(KW, 8)
    d = host.decode(KW, 32, maxpos=32, mmax=8)
    d.upload(P, stream)
    ok = np.arange(10, dtype=np.int32)
    d.sample_spec(ok, 23, stream)                         # the last position is 31
    for prompt, n, temp in ((ok, 24, 1.0), (ok, 0, 1.0), (ok[:0], 4, 1.0), (ok, 4, 0.0), (ok, 4, -1.0),
                            (ok, 4, float("nan")), (ok, 4, 1e30), (ok + 120, 4, 1.0), (ok - 1, 4, 1.0)):
        with pytest.raises(tlgemm.TlgError):
            d.sample_spec(prompt, n, stream, temp=temp)
    P[:] = np.nan                                          # no row has a distribution
    d.upload(P, stream)
    with pytest.raises(tlgemm.TlgError):
        d.sample_spec(ok, 4, stream)


def test_sample_spec_is_a_sample(lib, host, stream):
    """Second tokens over many seeds, kept drafts and others: their mean log
    probability is minus the entropy that the model gives, within 5 deviations."""
    kw = dict(KW, V=16, n_mtp=1)
    m, P = weights(kw, 9)
    d = host.decode(kw, 64, kv_f16=0, exact_exp=1, maxpos=64, mmax=4)
    d.upload(P, stream)
    prompt, temp = np.array([3, 1, 4], np.int32), 1.0
    runs = [d.sample_spec(prompt, 3, stream, temp=temp, seed=s)[:2] for s in range(400)]
    diffs = []
    for first in range(16):
        z = d.chunk(np.append(prompt, first).astype(np.int32), 0, stream)[3].astype(np.float64)
        lp = z - z.max() - np.log(np.exp(z - z.max()).sum())
        H, var = -(np.exp(lp) * lp).sum(), (np.exp(lp) * lp * lp).sum() - (np.exp(lp) * lp).sum() ** 2
        for toks, l in runs:
            if toks[0] == first:
                assert abs(l[1] - lp[toks[1]]) <= 1e-4
                diffs.append((l[1] + H, var))
    diffs = np.array(diffs)
    assert abs(diffs[:, 0].sum()) <= 5 * math.sqrt(diffs[:, 1].sum())
