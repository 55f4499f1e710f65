"""GPU tests of the serving operators (include/tlserve.h) against plain float64
evaluations of their definitions: rows into a paged cache, attention over it,
verification of drafts, and the three together.

Tolerances.  eps = 2^-24, half a step of fp32; half(type) that of a 16-bit type.
  store   a product and a fused or rounded product-sum: 3 eps (|a c| + |b s|), then
          the half step of what is written.
  attn    A score is a sum of hd products in any order, off by (hd + 1) eps
          sum_d |q_d k_d| scale, and its weight e^(s - m) by that, by the same of the
          maximum, by eps (4 |s - m| + 6) from the exponent and by half(type) for
          16-bit rows.  With d_t the sum of these, and n = L + 64 sequential additions at
          most in each sum, out is off by sum_t p_t |v_t| (2 d_t + 2 n eps) and its own
          half step, lse by the largest of d_t without half(type), + n eps + 2 eps |lse|.
  verify  whole numbers are equal: inputs are chosen away from borders (checked
          on the 64-bit side); logp as log probabilities: a weight is off by eps (4
          |z| + 6), a sum by that in the mean and its additions, chain(V) = 64 + V /
          64 at most.
"""
import math

import numpy as np
import pytest

import tlgemm

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
F32, F16, BF16 = 0, 1, 2
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
PAIRS = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
PAIR_IDS = [f"{NAMES[a]}-{NAMES[b]}" for a, b in PAIRS]


def _t():
    import torch
    return torch


@pytest.fixture(autouse=True)
def seeded():
    _t().manual_seed(0)


def dtype(ty):
    t = _t()
    return {F32: t.float32, F16: t.float16, BF16: t.bfloat16}[ty]


def half(ty):
    return {F32: EPS, F16: 2.0 ** -11, BF16: 2.0 ** -8}[ty]


def tiny(ty):
    return {F32: 2.0 ** -126, F16: 2.0 ** -25, BF16: 2.0 ** -126}[ty]


def stream():
    return _t().cuda.current_stream().cuda_stream


def ints(x):
    return _t().tensor(list(x), dtype=_t().int32).cuda()


class Seqs:
    """A batch with its paged cache.  rows and lens per sequence; pages dealt out
    at random; `head_major` puts [pages][KV][page][hd]; slots of no token hold NaN."""

    def __init__(self, rows, lens, KV, hd, page, kv, seed=0, head_major=False, extra_ldt=1, lead=0, tail=0, hints=True,
                 spare=1):
        t = _t()
        g = np.random.default_rng(seed)
        self.rows, self.lens, self.KV, self.hd, self.page, self.kv = rows, lens, KV, hd, page, kv
        self.lead, self.N, self.B = lead, lead + sum(rows) + tail, len(rows)
        need = [-(-max(n, 0) // page) for n in lens]
        self.n_pages, self.ldt = sum(need) + spare, max(need) + extra_ldt
        order = g.permutation(self.n_pages)
        self.table = np.full((self.B, self.ldt), -1, np.int64)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[at:at + k]
            at += k
        self.row0 = np.concatenate([[lead], lead + np.cumsum(rows)])
        shape = (self.n_pages, KV, page, hd) if head_major else (self.n_pages, page, KV, hd)
        self.head_major = head_major
        self.K = t.full(shape, float("nan"), dtype=dtype(kv))
        self.V = t.full(shape, float("nan"), dtype=dtype(kv))
        gen = t.Generator().manual_seed(seed)
        for b, n in enumerate(lens):
            if n > 0:
                for c in (self.K, self.V):
                    self.put(c, b, np.arange(n), t.randn(n, KV, hd, generator=gen).to(dtype(kv)))
        self.hints = hints
        self.max_rows, self.max_len = (max(rows), max(max(lens), 0)) if hints else (0, 0)

    def slots(self, b, pos):
        return _t().from_numpy(self.table[b][pos // self.page]), _t().from_numpy(pos % self.page)

    def put(self, c, b, pos, x):
        g, o = self.slots(b, pos)
        if self.head_major:
            c[g, :, o] = x
        else:
            c[g, o] = x

    def get(self, c, b, n):
        g, o = self.slots(b, np.arange(n))
        return (c[g, :, o] if self.head_major else c[g, o]).double()

    def gpu(self):
        t = _t()
        self.dK, self.dV = self.K.cuda(), self.V.cuda()
        self.dev = [ints(self.row0), ints(self.lens), t.from_numpy(self.table).int().cuda()]
        hm, p, d = self.head_major, self.page, self.hd
        self.pages = tlgemm.pages(self.dK.data_ptr(), self.dV.data_ptr(), self.kv, self.KV, d, p, self.n_pages,
                                  p * self.KV * d, d if hm else self.KV * d, p * d if hm else d)
        self.batch = tlgemm.batch(self.B, self.N, self.dev[0].data_ptr(), self.dev[1].data_ptr(), self.dev[2].data_ptr(),
                                  self.ldt, self.max_rows, self.max_len)
        return self


# ------------------------------------------------------------------- store --
def tables(maxpos, hd):
    a = np.arange(maxpos)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def ref_rope(x, pos, cs, sn):
    """x [n][heads][hd] float64 -> rotated, and the bound of the products' rounding."""
    h = x.shape[2] // 2
    ok = (pos >= 0) & (pos < len(cs))
    at = np.where(ok, pos, 0)
    c, s = cs[at][:, None].astype(np.float64), sn[at][:, None].astype(np.float64)
    c[~ok], s[~ok] = np.nan, np.nan
    a, b = x[..., :h], x[..., h:]
    out = np.concatenate([a * c - b * s, b * c + a * s], 2)
    mag = np.concatenate([abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)], 2)
    return out, 3 * EPS * mag


def check(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = np.broadcast_to(np.asarray(tol, np.float64), want.shape)
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), f"{what}: {np.isnan(got).sum()} NaN for {nan.sum()}"
    inf = np.isinf(want)
    assert (got[inf] == want[inf]).all(), what
    fin = ~(nan | inf)
    assert np.isfinite(got[fin]).all(), what
    err = abs(got - np.where(fin, want, 0.0))[fin]
    over = err - tol[fin]
    assert (over <= 0).all(), f"{what}: off by {err[over.argmax()]:.3g}, {tol[fin][over.argmax()]:.3g} allowed"


def run_store(lib, s, H, type, rope=True, maxpos=None, fused=False, inplace=False, use_q=True, q=None, seed=1):
    t = _t()
    KV, hd, N = s.KV, s.hd, s.N
    g = t.Generator().manual_seed(seed)
    wide = (H + 2 * KV) * hd
    x = t.randn(N, wide, generator=g).to(dtype(type)).cuda()
    parts = [x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]]
    if not fused:
        parts = [p.contiguous() for p in parts]
    want_in = [p.cpu().double().numpy() for p in parts]
    out = parts[0] if inplace else t.full((N, H * hd + 16), 7.0, dtype=dtype(type), device="cuda")[:, :H * hd]
    maxpos = max(s.lens) if maxpos is None else maxpos
    cs, sn = tables(max(maxpos, 1), hd)
    dc, ds = t.from_numpy(cs).cuda(), t.from_numpy(sn).cuda()
    lib.paged_store(s.pages, s.batch, parts[0].data_ptr() if use_q else None, parts[0].stride(0),
                    out.data_ptr() if use_q else None, out.stride(0), H, parts[1].data_ptr(), parts[1].stride(0),
                    parts[2].data_ptr(), parts[2].stride(0), type, dc.data_ptr() if rope else None,
                    ds.data_ptr() if rope else None, maxpos, stream())
    t.cuda.synchronize()
    return want_in, out, (cs[:maxpos], sn[:maxpos]) if rope else None


def check_store(s, H, type, want_in, out, cs, use_q=True, inplace=False, bad=()):
    KV, hd = s.KV, s.hd
    K, V = s.K.clone(), s.V.clone()
    q, k, v = want_in
    want_q = q.copy() if inplace else np.full(q.shape, 7.0)
    tol_q = np.zeros(q.shape)
    tolK = _t().zeros(K.shape, dtype=_t().float64)
    K64, V64 = K.double(), V.double()
    for b, (n, L) in enumerate(zip(s.rows, s.lens)):
        if n == 0:
            continue
        r0 = int(s.row0[b])
        pos = np.arange(L - n, L)

        def turn(x, heads):
            x = x[r0:r0 + n].reshape(n, heads, hd)
            return ref_rope(x, pos, *cs) if cs else (x, np.zeros(x.shape))
        o, e = turn(q, H)
        want_q[r0:r0 + n] = o.reshape(n, -1)
        tol_q[r0:r0 + n] = e.reshape(n, -1) + (half(type) * abs(o) + tiny(type)).reshape(n, -1) * (cs is not None)
        o, e = turn(k, KV)
        keep = (pos >= 0) & ~np.isin(np.maximum(pos, 0) // s.page, [p for bb, p in bad if bb == b])
        at = pos[keep]
        s.put(K64, b, at, _t().from_numpy(o[keep]))
        s.put(tolK, b, at, _t().from_numpy((e + half(s.kv) * abs(o) + tiny(s.kv))[keep]))
        s.put(V64, b, at, _t().from_numpy(v[r0:r0 + n].reshape(n, KV, hd)[keep]).to(dtype(s.kv)).double())
    if use_q:
        check(out.cpu().double().numpy(), want_q, tol_q, "q")
    check(s.dK.cpu().double().numpy(), K64.numpy(), tolK.numpy(), "K")
    check(s.dV.cpu().double().numpy(), V64.numpy(), 0.0, "V")


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows,lens,KV,H,hd,page,hm", [
    ([1], [1], 1, 1, 32, 1, False), ([1], [200], 3, 12, 32, 16, False), ([5, 0, 3, 1], [5, 9, 70, 33], 2, 4, 64, 7, True),
    ([17, 64], [17, 200], 1, 5, 96, 48, False), ([3] * 70, [40 + i for i in range(70)], 2, 2, 128, 16, True),
    ([9, 2], [30, 1000], 4, 4, 256, 64, False)])
def test_store(lib, type, kv, rows, lens, KV, H, hd, page, hm):
    s = Seqs(rows, lens, KV, hd, page, kv, head_major=hm, lead=2, tail=3).gpu()
    want, out, cs = run_store(lib, s, H, type, fused=hm)
    check_store(s, H, type, want, out, cs)


def test_store_without_rotation_or_queries(lib):
    for rope, use_q in ((False, True), (True, False), (False, False)):
        s = Seqs([4, 6], [4, 90], 2, 64, 16, BF16).gpu()
        want, out, cs = run_store(lib, s, 4, BF16, rope=rope, use_q=use_q)
        check_store(s, 4, BF16, want, out, cs, use_q=use_q)


def test_store_in_place(lib):
    s = Seqs([4, 6], [4, 90], 2, 64, 16, F16, lead=1, tail=2).gpu()
    want, out, cs = run_store(lib, s, 4, F16, inplace=True, fused=True)
    check_store(s, 4, F16, want, out, cs, inplace=True)


def test_store_at_positions_outside(lib):
    """Positions behind the tables are NaN; rows before position 0 and rows whose
    page is no page are not stored."""
    s = Seqs([6, 5, 4], [40, 3, 64], 2, 64, 16, F32).gpu()
    want, out, cs = run_store(lib, s, 2, F32, maxpos=37)
    check_store(s, 2, F32, want, out, cs)
    for number in (-1, -5, 10 ** 6, 2 ** 31 - 1):
        s = Seqs([6, 20], [40, 64], 2, 64, 16, F32)
        s.gpu()
        tab = s.dev[2].clone()
        tab[1, 3] = number
        s.dev[2].copy_(tab)
        want, out, cs = run_store(lib, s, 2, F32)
        check_store(s, 2, F32, want, out, cs, bad=[(1, 3)])


def test_store_table_too_short(lib):
    """Tokens behind the table's last column are not stored."""
    s = Seqs([8], [64], 1, 32, 16, F32).gpu()
    s.batch.ldt = 3                      # of one sequence: the same table, cut
    want, out, cs = run_store(lib, s, 2, F32)
    check_store(s, 2, F32, want, out, cs, bad=[(0, 3)])


# --------------------------------------------------------------- attention --
def ref_attn(s, q, H, type, scale, win, sinks, bad=()):
    """out, lse and their bounds, float64, for the rows of every sequence."""
    KV, hd = s.KV, s.hd
    G = H // KV
    out, lse = np.full((s.N, H, hd), np.nan), np.full((s.N, H), np.nan)
    tout, tlse = np.zeros((s.N, H, hd)), np.zeros((s.N, H))
    for b, (n, L) in enumerate(zip(s.rows, s.lens)):
        if n == 0:
            continue
        r0 = int(s.row0[b])
        pos, tt = np.arange(L - n, L)[:, None], np.arange(max(L, 0))[None]
        see = tt <= pos
        if win:
            see &= (tt > pos - win) | (tt < sinks)
        lost = np.isin(tt // s.page, [p for bb, p in bad if bb == b])
        k, v = s.get(s.K, b, max(L, 0)).numpy(), s.get(s.V, b, max(L, 0)).numpy()
        for h in range(H):
            qq, kk, vv = q[r0:r0 + n, h], k[:, h // G], v[:, h // G]
            with np.errstate(all="ignore"):
                z = np.where(see, scale * (qq @ kk.T), -np.inf)
                mag = np.where(see, scale * (abs(qq) @ abs(kk).T), 0.0)
                z = np.where(see & lost, np.nan, z)
                m = z.max(1, keepdims=True) if z.shape[1] else np.full((n, 1), -np.inf)
                e = np.where(see, np.exp(np.where(np.isneginf(m), 0.0, z - m)), 0.0)
                e = np.where(see & np.isneginf(z), 0.0, e)
                S = e.sum(1, keepdims=True)
                p = np.where(S == 0, 0.0, e / S)
                d = np.where(see, (hd + 1) * EPS * (mag + mag.max(1, keepdims=True, initial=0.0)) +
                             EPS * (4 * np.where(p > 0, abs(z - m), 0.0) + 6), 0.0)
                chain = EPS * (L + 64)
                out[r0:r0 + n, h] = [sum_rows(p[i], vv, see[i]) for i in range(n)]
                pv = np.array([sum_rows(p[i] * (2 * (d[i] + (half(type) if type else 0.0)) + 2 * chain), abs(vv), see[i])
                               for i in range(n)])
                o = out[r0:r0 + n, h]
                tout[r0:r0 + n, h] = pv + half(type) * abs(o) + tiny(type)
                ls = np.where(S[:, 0] == 0, -np.inf, m[:, 0] + np.log(S[:, 0]))
                lse[r0:r0 + n, h] = ls
                dm = np.where(see, d, 0.0).max(1, initial=0.0)
                tlse[r0:r0 + n, h] = dm + chain + 3 * EPS * np.where(np.isfinite(ls), abs(ls), 0.0)
    return out, lse, tout, tlse


def sum_rows(p, v, see):
    """sum_t p_t v_t over the tokens a row sees; the others' values may be anything."""
    return p[see] @ v[see] if see.any() else np.zeros(v.shape[1])


def run_attn(lib, s, q, H, type, scale, win=0, sinks=0, ldq=None, ldo=None, lse=True, fill=7.0, st=None):
    t = _t()
    ldq, ldo = ldq or H * s.hd, ldo or H * s.hd
    dq = t.full((s.N, ldq), float("nan"), dtype=dtype(type), device="cuda")
    dq[:, :H * s.hd] = q.reshape(s.N, -1).cuda()
    out = t.full((s.N, ldo), fill, dtype=dtype(type), device="cuda")
    ls = t.full((s.N, H), fill, device="cuda")
    nb = lib.paged_attn_ws_bytes(s.pages, s.batch, type, H)
    ws = t.full((nb + 4096,), 255, dtype=t.uint8, device="cuda")
    lib.paged_attn(s.pages, s.batch, dq.data_ptr(), type, ldq, H, scale, win, sinks, out.data_ptr(), ldo,
                   ls.data_ptr() if lse else None, ws.data_ptr() if nb else None, nb, stream() if st is None else st)
    t.cuda.synchronize()
    assert (ws[nb:] == 255).all(), "wrote behind its workspace"
    return out, ls


def queries(s, H, type, seed=3, spread=1.5):
    t = _t()
    return (spread * t.randn(s.N, H, s.hd, generator=t.Generator().manual_seed(seed))).to(dtype(type))


def check_attn(s, q, H, type, scale, win, sinks, out, ls, fill=7.0, bad=()):
    want, wl, to, tl = ref_attn(s, q.double().numpy(), H, type, scale, win, sinks, bad)
    inside = np.zeros(s.N, bool)
    inside[int(s.row0[0]):int(s.row0[-1])] = True
    o = out.cpu().double().numpy()
    width = H * s.hd
    assert (o[:, width:] == fill).all() and (o[~inside] == fill).all(), "wrote beside its rows"
    check(o[inside, :width].reshape(-1, H, s.hd), want[inside], to[inside], "out")
    if ls is not None:
        l = ls.cpu().double().numpy()
        assert (l[~inside] == fill).all()
        check(l[inside], wl[inside], tl[inside], "lse")


SHAPES = [
    # rows, lens, KV, H, hd, page, win, sinks
    ([1], [1], 1, 1, 32, 1, 0, 0),
    ([1], [250], 3, 12, 32, 16, 0, 0),
    ([1, 1, 0, 1, 1], [1, 33, 5, 64, 65], 2, 8, 64, 5, 0, 0),
    ([1] * 9, [7, 300, 31, 32, 127, 128, 129, 511, 1000], 1, 8, 128, 16, 0, 0),
    ([1, 1], [700, 90], 2, 2, 96, 48, 100, 3),
    ([1, 1], [513, 1500], 1, 16, 256, 64, 0, 0),
    ([5, 3, 0, 1, 4], [5, 400, 9, 77, 260], 2, 8, 64, 49, 64, 4),
    ([6], [900], 1, 40, 64, 32, 0, 0),
    ([33, 1, 70], [33, 200, 300], 2, 4, 64, 16, 0, 0),
    ([256], [256], 2, 8, 32, 32, 0, 0),
    ([130, 5], [400, 600], 1, 4, 128, 16, 90, 5),
    ([200], [333], 1, 3, 96, 7, 0, 0),
    ([65, 64], [65, 300], 1, 2, 256, 16, 31, 1),
    ([40], [40], 2, 2, 128, 128, 1, 0),
    ([50], [200], 1, 1, 64, 16, 8, 40),
]


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"rows{max(s[0])}-len{max(s[1])}-{s[2]}x{s[3]}x{s[4]}-p{s[5]}-w{s[6]}")
def test_attn(lib, type, kv, shape):
    rows, lens, KV, H, hd, page, win, sinks = shape
    s = Seqs(rows, lens, KV, hd, page, kv, head_major=page % 2 == 0, lead=1, tail=2).gpu()
    q = queries(s, H, type)
    out, ls = run_attn(lib, s, q, H, type, hd ** -0.5, win, sinks, ldq=H * hd + 16, ldo=H * hd + 8)
    check_attn(s, q, H, type, hd ** -0.5, win, sinks, out, ls)


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows,lens,win", [([1], [3000], 0), ([2, 40], [2500, 2600], 0), ([100], [4000], 3000)])
def test_attn_long(lib, type, kv, rows, lens, win):
    """Lengths whose keys are worked on in several places and joined."""
    s = Seqs(rows, lens, 1, 64, 16, kv).gpu()
    q = queries(s, 4, type)
    out, ls = run_attn(lib, s, q, 4, type, 0.125, win, 7 if win else 0)
    check_attn(s, q, 4, type, 0.125, win, 7 if win else 0, out, ls)


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows,lens", [([1, 3], [70, 200]), ([150], [300])])
def test_attn_hidden_values(lib, type, kv, rows, lens):
    """NaN and infinities in keys and values that a row does not see (later tokens
    of its chunk, tokens behind the window, free slots) do not reach it; those
    that it sees do."""
    t = _t()
    win, sinks = 40, 2
    s = Seqs(rows, lens, 1, 64, 16, kv)
    for b, (n, L) in enumerate(zip(rows, lens)):
        for c, val in ((s.K, float("nan")), (s.V, float("inf")), (s.V, float("nan"))):
            for pos in (L - 1, L - n // 2 - 1, max(L - n - win - 3, 3), 5 if L - n - win > 5 else L - 1):
                x = t.zeros(1, 1, 64, dtype=dtype(kv)) + 0.5
                x[..., 7] = val
                s.put(c, b, np.array([pos]), x)
    s.gpu()
    q = queries(s, 4, type)
    out, ls = run_attn(lib, s, q, 4, type, 0.125, win, sinks)
    check_attn(s, q, 4, type, 0.125, win, sinks, out, ls)


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows,lens", [([3, 5], [2, 5]), ([64, 9], [30, 0])])
def test_attn_rows_that_see_nothing(lib, type, kv, rows, lens):
    """Rows before position 0: 0, and -inf as their log-sum-exp."""
    s = Seqs(rows, lens, 1, 32, 4, kv).gpu()
    q = queries(s, 2, type)
    out, ls = run_attn(lib, s, q, 2, type, 0.2)
    check_attn(s, q, 2, type, 0.2, 0, 0, out, ls)
    assert (out.cpu()[0] == 0).all() and (ls.cpu()[0] == -math.inf).all()


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("number", [-1, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("rows,lens,win", [([1, 2], [70, 100], 0), ([90], [120], 0), ([90], [120], 20), ([1], [100], 20)])
def test_attn_bad_pages(lib, type, kv, number, rows, lens, win):
    """Rows that see a token without a page are NaN, the others as ever."""
    s = Seqs(rows, lens, 1, 64, 16, kv).gpu()
    b = len(rows) - 1
    s.dev[2][b, 3] = number
    q = queries(s, 2, type)
    out, ls = run_attn(lib, s, q, 2, type, 0.125, win)
    check_attn(s, q, 2, type, 0.125, win, 0, out, ls, bad=[(b, 3)])


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows,hd", [([2], 32), ([70], 128), ([3, 100], 64)])
def test_attn_cache_without_pages(lib, type, kv, rows, hd):
    """Nothing is read of it; rows that see a token are NaN, those before position 0 are 0.
    A store writes nothing there."""
    s = Seqs(rows, [30] * len(rows), 1, hd, 16, kv).gpu()
    s.pages.n_pages, s.pages.K, s.pages.V = 0, None, None
    for ldt in (s.ldt, 0):
        s.batch.ldt = ldt
        s.batch.table = s.dev[2].data_ptr() if ldt else None
        q = queries(s, 2, type)
        out, ls = run_attn(lib, s, q, 2, type, 0.2)
        o, l = out.cpu().float().numpy(), ls.cpu().numpy()
        for b, n in enumerate(rows):
            r = int(s.row0[b])
            before = max(n - 30, 0)
            assert (o[r:r + before] == 0).all() and np.isneginf(l[r:r + before]).all()
            assert np.isnan(o[r + before:r + n]).all() and np.isnan(l[r + before:r + n]).all()
        want, got, cs = run_store(lib, s, 2, type)
        assert np.isfinite(got.cpu().float().numpy()[max(rows) - 20:max(rows)]).all()


@pytest.mark.parametrize("type,kv", [(F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("rows,win", [([2], 0), ([90], 0), ([90], 10), ([1], 30)])
def test_attn_table_too_short(lib, type, kv, rows, win):
    s = Seqs(rows, [120], 1, 64, 16, kv).gpu()
    s.batch.ldt = 5                      # tokens from 80 on have no page
    q = queries(s, 2, type)
    out, ls = run_attn(lib, s, q, 2, type, 0.125, win)
    check_attn(s, q, 2, type, 0.125, win, 0, out, ls, bad=[(0, p) for p in range(5, 8)])


@pytest.mark.parametrize("type,kv", [(F32, F32), (F16, F16)])
def test_attn_wild_lengths(lib, type, kv):
    """Lengths far beyond the table or below zero end, in bounds."""
    s = Seqs([2, 3, 40], [50, 60, 70], 1, 32, 16, kv).gpu()
    q = queries(s, 2, type)
    s.dev[1].copy_(ints([2 ** 31 - 1, -7, 2 ** 30]))
    for win in (0, 9):
        out, ls = run_attn(lib, s, q, 2, type, 0.2, win)
        o = out.cpu().float().numpy()
        assert np.isnan(o[:2]).all() and (o[2:5] == 0).all() and np.isnan(o[5:]).all()
    s.dev[0].copy_(ints([-5, 10 ** 9, 3, 2]))            # rows out of order
    run_attn(lib, s, q, 2, type, 0.2)


@pytest.mark.parametrize("type,kv", [(F32, F16), (F16, F16), (BF16, BF16)])
def test_attn_hints_do_not_change_what_is_right(lib, type, kv):
    """Sequences longer and with more rows than the hints say, and no hints."""
    for hints in ((0, 0), (1, 10), (4, 4000), (300, 300), (1000, 0)):
        s = Seqs([150, 1, 7], [400, 1300, 60], 2, 64, 16, kv)
        s.max_rows, s.max_len = hints
        s.gpu()
        q = queries(s, 8, type)
        out, ls = run_attn(lib, s, q, 8, type, 0.125)
        check_attn(s, q, 8, type, 0.125, 0, 0, out, ls)


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
def test_attn_large_scores(lib, type, kv):
    """Scores far apart: one token takes it all, the rest underflow."""
    s = Seqs([1, 60], [200, 150], 1, 64, 16, kv).gpu()
    q = queries(s, 2, type, spread=30.0)
    for scale in (0.125, 2.0):
        out, ls = run_attn(lib, s, q, 2, type, scale)
        check_attn(s, q, 2, type, scale, 0, 0, out, ls)


def test_attn_same_bits_and_no_lse(lib):
    for rows, lens in (([1, 1], [2000, 300]), ([200, 3], [400, 900])):
        s = Seqs(rows, lens, 2, 64, 16, BF16).gpu()
        q = queries(s, 8, BF16)
        a, _ = run_attn(lib, s, q, 8, BF16, 0.125)
        for _ in range(3):
            b, l = run_attn(lib, s, q, 8, BF16, 0.125, lse=False)
            assert (a == b).all() and (l == 7.0).all()


def test_attn_many_sequences(lib):
    """More sequences than a wave has lanes, some without rows."""
    g = np.random.default_rng(5)
    rows = [int(x) for x in g.integers(0, 4, 150)]
    lens = [max(r, int(x)) for r, x in zip(rows, g.integers(1, 60, 150))]
    for type, kv in ((F32, F16), (BF16, BF16)):
        for hints in (True, False):
            s = Seqs(rows, lens, 1, 32, 8, kv, hints=hints, tail=4).gpu()
            q = queries(s, 4, type)
            out, ls = run_attn(lib, s, q, 4, type, 0.2)
            check_attn(s, q, 4, type, 0.2, 0, 0, out, ls)


@pytest.mark.parametrize("B", [130, 300, 1000, 1100])
def test_attn_many_sequences_with_room_for_long_ones(lib, B):
    """Tables that could hold more tokens than the sequences have, as a server's do:
    shares of the batch that span many short sequences, and a few long ones."""
    g = np.random.default_rng(B)
    rows = [int(x) for x in g.integers(0, 3, B)]
    lens = [max(r, int(x)) for r, x in zip(rows, g.integers(1, 50, B))]
    for b in (3, B // 2, B - 1):
        rows[b], lens[b] = 2, 1500 + b
    for type, kv, H in ((F32, F16, 2), (BF16, BF16, 12)):
        s = Seqs(rows, lens, 1, 32, 16, kv, hints=False, extra_ldt=60, lead=1).gpu()
        s.batch.max_rows = 2
        q = queries(s, H, type)
        out, ls = run_attn(lib, s, q, H, type, 0.2)
        check_attn(s, q, H, type, 0.2, 0, 0, out, ls)


@pytest.mark.parametrize("type,kv", [(F32, F32), (F16, F16)])
@pytest.mark.parametrize("rows,H,hd", [([1], 2, 32), ([9, 0, 1], 3, 64)])
def test_attn_hundreds_of_shares(lib, type, kv, rows, H, hd):
    """One long sequence that every workgroup takes a part of."""
    s = Seqs(rows, [66001] + [5] * (len(rows) - 1), 1, hd, 64, kv).gpu()
    q = queries(s, H, type)
    out, ls = run_attn(lib, s, q, H, type, hd ** -0.5)
    check_attn(s, q, H, type, hd ** -0.5, 0, 0, out, ls)


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("hd", [96, 128, 256])
def test_attn_shares_of_wide_heads(lib, type, kv, hd):
    """Ragged lengths shared evenly, in blocks of 16 and of 32 columns."""
    for rows, H in (([1, 2, 1], 4), ([3, 1, 6], 4)):
        s = Seqs(rows, [2600, 90, 700], 1, hd, 16, kv, head_major=True).gpu()
        q = queries(s, H, type)
        out, ls = run_attn(lib, s, q, H, type, hd ** -0.5)
        check_attn(s, q, H, type, hd ** -0.5, 0, 0, out, ls)


@pytest.mark.parametrize("page", [16, 48, 33])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_attn_long_chunks_of_two_layouts(lib, page, hd):
    """Many 16-bit rows: pages that a wave's load does and does not stay within, in
    both layouts, a chunk in the middle of a page."""
    for hm in (True, False):
        s = Seqs([100, 45], [391, 300], 2, hd, page, BF16, head_major=hm).gpu()
        q = queries(s, 6, BF16)
        out, ls = run_attn(lib, s, q, 6, BF16, hd ** -0.5, 150, 20)
        check_attn(s, q, 6, BF16, hd ** -0.5, 150, 20, out, ls)


def test_attn_pages_far_apart(lib):
    """Offsets beyond 2^32 elements: pages in a buffer with large gaps."""
    t = _t()
    s = Seqs([2, 40], [40, 90], 1, 64, 16, F16)
    s.gpu()
    gap = (1 << 32) // s.n_pages // 8 * 8 + 4096
    bufs = []
    for c in (s.K, s.V):
        buf = t.empty(gap * (s.n_pages - 1) + 16 * 64, dtype=t.float16, device="cuda")
        t.as_strided(buf, (s.n_pages, 16, 64), (gap, 64, 1)).copy_(c.reshape(s.n_pages, 16, 64).cuda())
        bufs.append(buf)
    s.pages.K, s.pages.V, s.pages.page_ld = bufs[0].data_ptr(), bufs[1].data_ptr(), gap
    q = queries(s, 2, F16)
    out, ls = run_attn(lib, s, q, 2, F16, 0.125)
    check_attn(s, q, 2, F16, 0.125, 0, 0, out, ls)


@pytest.mark.parametrize("type,kv", [(F32, F16), (BF16, BF16)])
def test_attn_captured_while_lengths_grow(lib, type, kv):
    """A captured step replays at the lengths that it finds, on a stream of its
    own, with eager work between the replays."""
    t = _t()
    s = Seqs([1, 1, 2], [300, 40, 700], 1, 64, 16, kv)
    s.max_len = 1000
    s.gpu()
    H = 4
    q = queries(s, H, type)
    dq = q.reshape(s.N, -1).cuda()
    out, ls = t.zeros(s.N, H * 64, dtype=dtype(type), device="cuda"), t.zeros(s.N, H, device="cuda")
    nb = lib.paged_attn_ws_bytes(s.pages, s.batch, type, H)
    ws = t.empty(max(nb, 16), dtype=t.uint8, device="cuda")
    st = lib.tlg_stream_create()
    lib.check(lib.tlg_graph_begin(st))
    lib.paged_attn(s.pages, s.batch, dq.data_ptr(), type, H * 64, H, 0.125, 0, 0, out.data_ptr(), H * 64, ls.data_ptr(),
                   ws.data_ptr(), nb, st)
    g = lib.tlg_graph_end(st)
    assert g
    lens = list(s.lens)
    for step in range(4):
        s.lens = [l - 5 * step for l in lens]
        s.dev[1].copy_(ints(s.lens))
        out.fill_(7.0)
        t.cuda.synchronize()
        lib.check(lib.tlg_graph_launch(g, st))
        lib.check(lib.tlg_stream_sync(st))
        check_attn(s, q, H, type, 0.125, 0, 0, out, ls)
        again, l2 = run_attn(lib, s, q, H, type, 0.125)
        assert (again == out).all() and (l2 == ls).all()
    lib.tlg_graph_destroy(g)
    lib.tlg_stream_destroy(st)


def test_two_streams_at_once(lib):
    """Calls with their own outputs and workspaces overlap."""
    t = _t()
    sets = []
    for i, type in enumerate((BF16, F32)):
        s = Seqs([1, 60], [1500, 200 + i], 1, 64, 16, BF16 if type else F16, seed=i).gpu()
        q = queries(s, 4, type)
        nb = lib.paged_attn_ws_bytes(s.pages, s.batch, type, 4)
        sets.append((s, q, type, q.reshape(s.N, -1).cuda(), t.empty(s.N, 256, dtype=dtype(type), device="cuda"),
                     t.empty(s.N, 4, device="cuda"), t.empty(max(nb, 16), dtype=t.uint8, device="cuda"), nb,
                     t.cuda.Stream()))
    t.cuda.synchronize()
    for _ in range(5):
        for s, q, type, dq, out, ls, ws, nb, st in sets:
            lib.paged_attn(s.pages, s.batch, dq.data_ptr(), type, 256, 4, 0.125, 0, 0, out.data_ptr(), 256, ls.data_ptr(),
                           ws.data_ptr(), nb, st.cuda_stream)
    t.cuda.synchronize()
    for s, q, type, dq, out, ls, ws, nb, st in sets:
        check_attn(s, q, 4, type, 0.125, 0, 0, out, ls)


# ------------------------------------------------------------------ verify --
def log_softmax(x, scale):
    """x [n][V] float64; rows of nothing but -inf give -inf, with NaN or +inf NaN."""
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        z = np.where(np.isneginf(m), -np.inf, (x - m) * scale)
        return np.where(np.isneginf(m), -np.inf, z - np.log(np.exp(z).sum(1, keepdims=True)))


def ref_verify(x, y, row0, draft, u, e, scale, dscale, border=1e-5):
    """tokens, logp, accepted; asserts that no decision lies near its border."""
    N, V = x.shape
    B = len(row0) - 1
    tokens, logp, acc = np.full(N, -9), np.full(N, np.nan), np.zeros(B, np.int64)
    lp = log_softmax(x, scale)
    lq = None if y is None else log_softmax(y, dscale)
    for b in range(B):
        lo, hi = row0[b], row0[b + 1]
        tokens[lo:hi], logp[lo:hi] = -1, 0.0
        for r in range(lo, hi):
            d = draft[r] if r < hi - 1 else -1
            pr, pick, refused = lp[r], False, False
            with np.errstate(all="ignore"):
                if np.isnan(pr).any() or np.isneginf(pr).all():
                    logp[r] = np.nan
                    break
                if d >= 0:
                    if lq is not None and np.isnan(lq[r]).any():
                        logp[r] = np.nan
                        break
                    pd = pr[d] if d < V else -np.inf
                    qd = 0.0 if lq is None else lq[r][d] if d < V else -np.inf
                    left, right = u[r] * np.exp(qd), np.exp(pd)
                    assert left == right == 0 or abs(left - right) > border * max(left, right), "a test at its border"
                    if left < right:
                        tokens[r], logp[r] = d, pd
                        acc[b] += 1
                        continue
                    refused = True
                w = np.exp(pr)
                if refused:
                    w2 = w.copy()
                    if lq is None:
                        if d < V:
                            w2[d] = 0.0
                    else:
                        w2 = np.maximum(0.0, w2 - np.exp(lq[r]))
                    if (w2 > 1e-12).any():
                        w = w2
                ok = (e[b] >= 1e-30) & (e[b] <= 1e30)
                k = np.where(ok, w / np.where(ok, e[b], 1.0), 0.0)
            if not (k > 0).any():
                logp[r] = np.nan
                break
            v = int(k.argmax())
            rest = np.delete(k, v)
            if len(rest):
                assert rest.max() < k[v] * (1 - border) or rest.max() == k[v], "a race at its border"
            tokens[r], logp[r] = v, pr[v]
            break
    return tokens, logp, acc


class Drafts:
    def __init__(self, rows, V, type, drafted=True, seed=0, pad=0, off=0, lead=0, tail=0, spread=2.0, scale=1.0, dscale=1.0,
                 agree=0.5):
        t = _t()
        self.rows, self.V, self.type, self.scale, self.dscale = rows, V, type, scale, dscale
        self.B, self.N = len(rows), lead + sum(rows) + tail
        self.row0 = np.concatenate([[lead], lead + np.cumsum(rows)]).astype(np.int64)
        g = t.Generator().manual_seed(seed)
        ld = V + pad

        def rows_of(v):
            buf = t.full((off + self.N * ld + 16,), float("nan"), dtype=dtype(type))
            x = t.as_strided(buf, (self.N, V), (ld, 1), off)
            x.copy_(v.to(dtype(type)))
            return [buf, x]
        base = spread * t.randn(self.N, V, generator=g)
        base[:, :3] += 4.0
        self.x = rows_of(base)
        self.y = rows_of(base + agree * t.randn(self.N, V, generator=g)) if drafted else None
        self.u = t.rand(self.N, generator=g)
        self.e = t.empty(self.B, V).exponential_(generator=g).clamp_min_(1e-9)
        pick = (self.y or self.x)[1].float() * dscale
        self.draft = (pick - t.empty(self.N, V).exponential_(generator=g).log()).argmax(1).int()

    def ref(self, border=1e-5):
        return ref_verify(self.x[1].double().numpy(), None if self.y is None else self.y[1].double().numpy(), self.row0,
                          self.draft.numpy(), self.u.double().numpy(), self.e.double().numpy(), self.scale, self.dscale,
                          border)

    def run(self, lib, logp=True, accepted=True, st=None):
        t = _t()

        def put(p):
            b = p[0].cuda()
            return b, t.as_strided(b, p[1].shape, p[1].stride(), p[1].storage_offset())
        bx, x = put(self.x)
        by, y = put(self.y) if self.y else (None, None)
        dev = [ints(self.row0), self.draft.cuda(), self.u.cuda(), self.e.cuda()]
        tok = t.full((self.N,), -9, dtype=t.int32, device="cuda")
        lp = t.full((self.N,), 9.0, device="cuda")
        acc = t.full((self.B,), -9, dtype=t.int32, device="cuda")
        nb = lib.tlg_spec_verify_ws_bytes(self.type, self.N, self.V, self.B, int(self.y is not None))
        ws = t.full((max(nb, 16),), 255, dtype=t.uint8, device="cuda")
        lib.spec_verify(x.data_ptr(), self.type, x.stride(0), self.scale, y.data_ptr() if self.y else None,
                        y.stride(0) if self.y else 0, self.dscale, self.N, self.V, dev[0].data_ptr(), self.B,
                        dev[1].data_ptr(), dev[2].data_ptr(), dev[3].data_ptr(), self.e.shape[1], tok.data_ptr(),
                        lp.data_ptr() if logp else None, acc.data_ptr() if accepted else None, ws.data_ptr(), nb,
                        stream() if st is None else st)
        t.cuda.synchronize()
        return tok.cpu().numpy(), lp.cpu().numpy(), acc.cpu().numpy()

    def check(self, got, border=1e-5):
        tok, lp, acc = self.ref(border)
        assert (got[0] == tok).all(), (got[0][got[0] != tok], tok[got[0] != tok])
        assert (got[2] == acc).all()
        inside = np.zeros(self.N, bool)
        inside[self.row0[0]:self.row0[-1]] = True
        assert (got[1][~inside] == 9.0).all()
        lv = math.log(self.V + 1)
        z = np.where(np.isfinite(lp), abs(lp), 0.0)
        tol = EPS * (4 * z + 6 + 4 * lv + 6 + 64 + self.V / 64 + 2 * z)
        check(got[1][inside], lp[inside], tol[inside], "logp")


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("rows,V,pad,off", [([3], 2048, 0, 0), ([1], 1, 0, 0), ([2, 0, 5, 1], 7, 3, 1),
                                            ([4, 4, 4], 1003, 0, 3), ([5] * 20, 5021, 11, 2), ([9], 131072, 0, 0),
                                            ([1, 2], 131071, 1, 5), ([6, 300], 65, 0, 1)])
def test_verify(lib, type, drafted, rows, V, pad, off):
    d = Drafts(rows, V, type, drafted, seed=V + off, pad=pad, off=off, lead=1, tail=2, scale=0.8, dscale=1.25)
    d.check(d.run(lib))


@pytest.mark.parametrize("type", [F32, BF16])
def test_verify_keeps_all_and_none(lib, type):
    d = Drafts([5, 5], 300, type, True, seed=2)
    d.u.fill_(0.0)
    got = d.run(lib)
    d.check(got)
    assert (got[2] == 4).all()
    d.draft[:] = 250
    d.x[1][:, 250] = -20.0
    d.y[1][:, 250] = 20.0
    d.u.fill_(0.5)
    got = d.run(lib)
    d.check(got)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("drafted", [True, False])
def test_verify_rows_without_a_distribution(lib, type, drafted):
    """Masked tokens, rows of nothing but -inf, NaN and +inf in either row, drafts
    out of range or missing, one token left."""
    inf, nan = math.inf, math.nan
    d = Drafts([4] * 10, 130, type, drafted, seed=4)
    x, y = d.x[1], d.y[1] if drafted else None
    d.u.fill_(1e-3)
    row = lambda b, i: int(d.row0[b]) + i
    x[row(0, 1), :] = -inf
    x[row(1, 1), 129] = nan
    x[row(2, 2), 128] = inf
    d.draft[row(3, 1)] = -1
    d.draft[row(4, 1)] = 130
    d.draft[row(5, 0)] = 2 ** 31 - 1
    x[row(6, 0), 10:] = -inf
    d.draft[row(6, 0)] = 77                       # a masked draft
    x[row(7, 0), :] = -inf
    x[row(7, 0), 5] = 0.0
    d.draft[row(7, 0)] = 5
    x[row(7, 1), :] = -inf
    x[row(7, 1), 6] = -3.0
    d.draft[row(7, 1)] = 9
    if drafted:
        y[row(8, 0), :] = -inf                    # q = 0: kept where p > 0
        y[row(8, 1), 3] = nan
        y[row(9, 3), 3] = nan                     # the last row has no draft: not looked at
        y[row(9, 0), 3] = inf
    d.check(d.run(lib))


@pytest.mark.parametrize("type", [F32, BF16])
def test_verify_noise(lib, type):
    """Noise outside its range is not chosen; equal keys go to the lowest token."""
    d = Drafts([1] * 6, 700, type, True, seed=6)
    d.e[0, :3] = 0.0
    d.e[1, :3] = math.nan
    d.e[2, :3] = -1.0
    d.e[3, :] = 0.0
    d.e[4, :] = math.inf
    d.x[1][5, :] = 1.0
    d.e[5, :] = 2.0
    d.e[5, 300:] = 1.0
    got = d.run(lib)
    d.check(got)
    assert got[0][5] == 300 and got[0][3] == -1 and got[0][4] == -1


@pytest.mark.parametrize("type", [F32, F16, BF16])
def test_verify_far_logits(lib, type):
    """Logits and scales far apart."""
    d = Drafts([3, 3], 500, type, True, seed=8)
    big = 3e4 if type == F16 else 1e30
    d.x[1][0, :] -= big
    d.x[1][1, 4] = -big
    d.y[1][1, 5] = -big
    d.check(d.run(lib))
    d = Drafts([3, 3], 500, type, False, seed=9, scale=1e4)
    d.check(d.run(lib))
    d = Drafts([3, 3], 500, type, True, seed=9, scale=1e-20, dscale=1e-20)
    d.y[1].copy_(d.x[1])
    d.u.fill_(0.5)
    d.check(d.run(lib), border=0.0 if type else 1e-7)


def test_verify_optional_outputs_and_same_bits(lib):
    d = Drafts([5, 2, 0, 8], 40000, BF16, True, seed=3)
    a = d.run(lib)
    d.check(a)
    b = d.run(lib, logp=False, accepted=False)
    assert (b[0] == a[0]).all() and (b[1] == 9.0).all() and (b[2] == -9).all()
    c = d.run(lib)
    assert all((p == q).all() for p, q in zip(a, c))


def test_verify_no_rows(lib):
    d = Drafts([0, 0, 0], 50, F32, True)
    t = _t()
    acc = t.full((3,), -9, dtype=t.int32, device="cuda")
    r0 = ints([0, 0, 0, 0])
    lib.spec_verify(None, F32, 50, 1.0, None, 50, 1.0, 0, 50, r0.data_ptr(), 3, None, None, None, 50, None, None,
                    acc.data_ptr(), None, 0, stream())
    assert (acc.cpu() == 0).all()


def test_verify_wild_rows(lib):
    """Row numbers out of range or order stay in bounds."""
    d = Drafts([3, 3, 3], 100, F32, True)
    for row0 in ([-4, 3, 100, 10 ** 9], [9, 6, 3, 0], [0, 0, 9, 9]):
        d.row0 = np.array(row0)
        tok, _, acc = d.run(lib)
        assert ((tok >= -9) & (tok < 100)).all() and ((acc >= 0) & (acc <= 9)).all()


def test_verify_replayed(lib):
    """Captured once, replayed with other numbers in the same buffers."""
    t = _t()
    d = Drafts([4, 4, 1], 9000, F16, True, seed=1)
    x, y = d.x[1].cuda(), d.y[1].cuda()
    dev = [ints(d.row0), d.draft.cuda(), d.u.cuda(), d.e.cuda()]
    tok, acc = t.zeros(d.N, dtype=t.int32, device="cuda"), t.zeros(d.B, dtype=t.int32, device="cuda")
    lp = t.zeros(d.N, device="cuda")
    nb = lib.tlg_spec_verify_ws_bytes(F16, d.N, d.V, d.B, 1)
    ws = t.empty(nb, dtype=t.uint8, device="cuda")
    st = lib.tlg_stream_create()
    lib.check(lib.tlg_graph_begin(st))
    lib.spec_verify(x.data_ptr(), F16, x.stride(0), 1.0, y.data_ptr(), y.stride(0), 1.0, d.N, d.V, dev[0].data_ptr(), d.B,
                    dev[1].data_ptr(), dev[2].data_ptr(), dev[3].data_ptr(), d.V, tok.data_ptr(), lp.data_ptr(),
                    acc.data_ptr(), ws.data_ptr(), nb, st)
    g = lib.tlg_graph_end(st)
    for i in range(4):
        n = Drafts([4, 4, 1], 9000, F16, True, seed=20 + i)
        x.copy_(n.x[1])
        y.copy_(n.y[1])
        for a, b in zip(dev[1:], (n.draft, n.u, n.e)):
            a.copy_(b)
        t.cuda.synchronize()
        lib.check(lib.tlg_graph_launch(g, st))
        lib.check(lib.tlg_stream_sync(st))
        n.check((tok.cpu().numpy(), lp.cpu().numpy(), acc.cpu().numpy()))
    lib.tlg_graph_destroy(g)
    lib.tlg_stream_destroy(st)


def test_verify_distribution(lib):
    """The first token given back is a sample of p, whatever the draft model: counts
    of 40000 sequences against p, each within 5 deviations of a binomial count."""
    t = _t()
    V, n = 12, 40000
    g = t.Generator().manual_seed(11)
    lx, ly = 1.5 * t.randn(V, generator=g), 1.5 * t.randn(V, generator=g)
    for drafted in (True, False):
        d = Drafts([2] * n, V, F32, drafted, seed=12)
        d.x[1].copy_(lx.expand(2 * n, V))
        if drafted:
            d.y[1].copy_(ly.expand(2 * n, V))
            d.draft = (ly - t.empty(2 * n, V).exponential_(generator=g).log()).argmax(1).int()
        else:
            d.draft.fill_(4)
        tok, _, _ = d.run(lib)
        p = t.softmax(lx.double(), 0).numpy()
        got = np.bincount(tok[0::2], minlength=V)
        assert (abs(got - n * p) <= 5 * np.sqrt(n * p * (1 - p)) + 1).all(), (got, n * p)
