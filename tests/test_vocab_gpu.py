"""GPU tests of the operators over rows of logits (include/tltrain.h): log
probabilities with entropy and alternatives, their gradient, distillation,
against plain float64 evaluations of their definitions.

Tolerances.  eps = 2^-24, half a step of fp32.  An exponential e^z', z' = s (x -
m), is formed from the rounded difference, a product with a rounded constant
and a hardware exponential of one unit in the last place: relative error
<= eps (4 |z'| + 3).  A sum of a row runs over at most C(V) = 64 + V / 256
sequential fp32 additions, rescalings among them, each off by eps at most.  With
weights p the mean |z'| is entropy - log S <= log V, so S is off by rho = eps (4
log V + 3 + C) relative and log S by rho + 2 eps |log S| absolute.  The other
bounds follow from these term by term, as written at each check.  Outputs in
fp16 or bf16 add the half step of their type (fp16 below its normal range
2^-25 absolute).
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
F32, F16, BF16 = 0, 1, 2
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}


def _t():
    import torch
    return torch


@pytest.fixture(autouse=True)
def seeded():
    """The same inputs on every run and in every selection of tests: torch seeds
    the GPU's generator by chance."""
    _t().manual_seed(0)


def dtype(ty):
    t = _t()
    return {F32: t.float32, F16: t.float16, BF16: t.bfloat16}[ty]


def half_step(ty):
    return {F32: EPS, F16: 2.0 ** -11, BF16: 2.0 ** -8}[ty]


def tiny(ty):
    """Half the smallest step of the type, where relative bounds end."""
    return {F32: 2.0 ** -126, F16: 2.0 ** -25, BF16: 2.0 ** -126}[ty]


def stream():
    return _t().cuda.current_stream().cuda_stream


def chain(V):
    return 64 + V / 256


def rho(V):
    return EPS * (4 * math.log(V + 1) + 3 + chain(V))


def rows_of(ty, N, V, ld=None, off=0, seed=0, spread=2.5, fill=float("nan")):
    """Logits [N][V] in rows ld apart that start `off` elements into a buffer,
    with `fill` between and around them."""
    t = _t()
    ld = ld or V
    g = t.Generator().manual_seed(seed + 7919 * V + N)
    buf = t.full((off + N * ld + 16,), fill, dtype=dtype(ty))
    x = t.as_strided(buf, (N, V), (ld, 1), off)
    x.copy_((spread * t.randn(N, V, generator=g)).to(dtype(ty)))
    return buf, (N, V), (ld, 1), off


def on_gpu(rows):
    buf, shape, strides, off = rows
    b = buf.cuda()
    return b, _t().as_strided(b, shape, strides, off)


def like_rows(x, ty, fill=float("nan")):
    """A gradient buffer of x's layout, filled."""
    t = _t()
    b = t.full((x.storage_offset() + x.shape[0] * x.stride(0) + 16,), fill, dtype=dtype(ty), device="cuda")
    return b, t.as_strided(b, tuple(x.shape), (x.stride(0), 1), x.storage_offset())


def f64(x):
    return x.detach().cpu().double().numpy()


# ------------------------------------------------------------- definitions --
def ref_logp(x, scale):
    """x [N][V] float64 -> (log probabilities, m, log S, entropy)."""
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        z = np.where(np.isneginf(m), -np.inf, (x - m) * scale)
        z[np.isnan(x)] = np.nan
        S = np.exp(z).sum(1, keepdims=True)
        lp = z - np.log(S)
        lp[np.isneginf(m[:, 0])] = -np.inf
        p = np.exp(lp)
        H = -np.where(p > 0, p * lp, 0.0).sum(1)
        H = np.where(np.isnan(S[:, 0]), np.nan, H)
    return lp, m[:, 0], np.log(S[:, 0]), H


def ref_top(x, K):
    """The K largest unmasked values of every row, the lower index first among
    equals; -1 where fewer are left."""
    out = np.full((x.shape[0], K), -1, np.int64)
    for n, row in enumerate(x):
        order = np.argsort(-row, kind="stable")
        order = order[row[order] > -np.inf][:K]
        out[n, :len(order)] = order
    return out


def ref_bwd(x, scale, ids, dlogp, dlse, dent):
    lp, _, _, H = ref_logp(x, scale)
    p = np.exp(lp)
    d = p * (dlse - np.where(ids >= 0, dlogp, 0.0).sum(1))[:, None]
    d -= dent[:, None] * np.where(p > 0, p * (np.where(p > 0, lp, 0.0) + H[:, None]), 0.0)
    for n in range(x.shape[0]):
        if np.isneginf(x[n]).all():
            continue
        for j, i in enumerate(ids[n]):
            if i >= 0:
                d[n, i] += dlogp[n, j]
    return d * scale


def ref_distill(x, ids, tl, tail, tau, w_kd, tgt, w_ce):
    """(rows, d rows / d x) in float64."""
    N, V = x.shape
    rows, grad = np.zeros(N), np.zeros((N, V))
    lp, lp1 = ref_logp(x, 1.0 / tau)[0], ref_logp(x, 1.0)[0]
    for n in range(N):
        q, seen = np.zeros(V), np.zeros(V, bool)
        for i, l in zip(ids[n], tl[n]):
            if i >= 0 and not seen[i]:
                seen[i], q[i] = True, math.exp(l)
        p = np.exp(lp[n])
        qr = 0.0
        if not tail:
            q = q / q.sum() if q.sum() > 0 else q
        elif seen.any() and not seen.all():
            qr = max(0.0, 1.0 - q.sum())
        on = q > 0
        kl = (q[on] * (np.log(q[on]) - lp[n][on])).sum()
        mass = (q.sum() + qr) * np.ones(V)
        if qr > 0:
            pr = p[~seen].sum()
            with np.errstate(all="ignore"):
                kl += qr * (math.log(qr) - np.log(pr))
                mass[~seen] = (q.sum() + qr) - (qr / pr if pr > 0 else 0.0)
        rows[n] = w_kd * tau * tau * kl
        grad[n] = w_kd * tau * (mass * p - q)
        if w_ce and tgt[n] >= 0:
            rows[n] -= w_ce * lp1[n, tgt[n]]
            grad[n] += w_ce * np.exp(lp1[n])
            grad[n, tgt[n]] -= w_ce
    return rows, grad


# ------------------------------------------------------------------- calls --
class Out:
    pass


def logprobs(lib, x, ty, scale, ids, K, ws_fill=255):
    t = _t()
    N, V = x.shape
    o = Out()
    M = 0 if ids is None else ids.shape[1]
    nan = float("nan")
    o.logp = t.full((N, M), nan, device="cuda")
    o.lse2 = t.full((N, 2), nan, device="cuda")
    o.entropy = t.full((N,), nan, device="cuda")
    o.top_ids = t.full((N, K), -77, device="cuda", dtype=t.int32)
    o.top_logp = t.full((N, K), nan, device="cuda")
    nb = lib.tlg_logprobs_ws_bytes(ty, N, V, K)
    o.ws = t.full((nb + 16,), ws_fill, device="cuda", dtype=t.uint8)
    lib.logprobs(x.data_ptr(), ty, x.stride(0), N, V, scale, ids.data_ptr() if M else None, M, o.logp.data_ptr(),
                 o.lse2.data_ptr(), o.entropy.data_ptr(), K, o.top_ids.data_ptr(), o.top_logp.data_ptr(),
                 o.ws.data_ptr(), nb, stream())
    return o


def logprobs_bwd(lib, x, ty, scale, ids, lse2, entropy, dlogp, dlse, dent, d):
    M = 0 if ids is None else ids.shape[1]

    def p(v):
        return None if v is None else v.data_ptr()
    lib.logprobs_bwd(x.data_ptr(), ty, x.stride(0), x.shape[0], x.shape[1], scale, p(ids), M, p(lse2), p(entropy),
                     p(dlogp), p(dlse), p(dent), d.data_ptr(), d.stride(0), stream())


def distill(lib, x, ty, t_ids, t_logp, tail, tau, w_kd, tgt, w_ce, d, scale=1.0, ws_fill=255):
    t = _t()
    N, V = x.shape
    K = 0 if t_ids is None else t_ids.shape[1]
    o = Out()
    o.rows = t.full((N,), float("nan"), device="cuda")
    o.loss = t.full((1,), float("nan"), device="cuda")
    nb = lib.tlg_distill_ws_bytes(ty, N, V)
    o.ws = t.full((nb + 16,), ws_fill, device="cuda", dtype=t.uint8)
    lib.distill(x.data_ptr(), ty, x.stride(0), N, V, t_ids.data_ptr() if K else None,
                t_logp.data_ptr() if K else None, K, int(tail), tau, w_kd, None if tgt is None else tgt.data_ptr(),
                w_ce, o.rows.data_ptr(), o.loss.data_ptr(), None if d is None else d.data_ptr(),
                0 if d is None else d.stride(0), scale, o.ws.data_ptr(), nb, stream())
    return o


# ------------------------------------------------------------------ checks --
def close(got, want, tol, what):
    """got within tol of want element by element; infinities and NaN equal."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), what
    err, bar = np.abs(got - want)[fin], np.broadcast_to(tol, want.shape)[fin]
    if err.size:
        k = int(np.argmax(err - bar))
        assert (err <= bar).all(), (what, "worst", err[k], "allowed", bar[k])


def check_logprobs(o, x, scale, ids, K):
    X = f64(x)
    V = X.shape[1]
    lp, m, ls, H = ref_logp(X, scale)
    bad = np.isnan(ls)
    tol_ls = rho(V) + 2 * EPS * np.abs(np.where(np.isfinite(ls), ls, 0.0))
    close(f64(o.lse2)[:, 0], np.where(bad, np.nan, m), 0.0, "max")
    close(f64(o.lse2)[:, 1], np.where(np.isneginf(m), -np.inf, ls), tol_ls, "log sum")

    def tol_lp(v):       # two roundings of z', log S, the final one
        v = np.where(np.isfinite(v), np.abs(v), 0.0)
        return 4 * EPS * (v + np.abs(np.where(np.isfinite(ls), ls, 0.0))[:, None]) + tol_ls[:, None]
    if ids is not None and ids.shape[1]:
        I = ids.cpu().numpy()
        want = np.take_along_axis(lp, np.clip(I, 0, V - 1), 1)
        want = np.where(I < 0, 0.0, np.where(I >= V, np.nan, want))
        close(f64(o.logp), want, tol_lp(want), "logp")
    # H = log S - u / S, both sums rho-close; |u / S| <= log V
    lv = math.log(V + 1)
    tol_H = tol_ls + 2 * (rho(V) + 4 * EPS) * lv + 2 * EPS * np.abs(np.where(np.isfinite(H), H, 0.0))
    close(f64(o.entropy), np.where(np.isneginf(m), 0.0, H), tol_H, "entropy")
    if K:
        top = ref_top(X, K)
        top[bad] = -1
        assert np.array_equal(o.top_ids.cpu().numpy(), top), "top ids"
        want = np.where(top < 0, -np.inf, np.take_along_axis(lp, np.clip(top, 0, V - 1), 1))
        want[bad] = np.nan
        close(f64(o.top_logp), want, tol_lp(want), "top logp")


def some_ids(N, V, M, seed, none=True):
    t = _t()
    g = t.Generator().manual_seed(seed)
    ids = t.randint(0, V, (N, M), generator=g, dtype=t.int32)
    if none and N > 1:
        ids[N // 2, 0] = -1
    return ids.cuda()


SIZES = [(1, 1, 1), (3, 2, 2), (2, 3, 5), (5, 7, 4), (4, 31, 40), (3, 64, 64), (9, 65, 8), (2, 255, 128), (3, 257, 20),
         (5, 1000, 16), (7, 2047, 33), (130, 2048, 8), (3, 2049, 128), (2, 4097, 60), (6, 8191, 5), (1, 16384, 128),
         (3, 32003, 32), (1, 65537, 20), (2, 131072, 100)]


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("N,V,K", SIZES)
def test_logprobs(lib, ty, N, V, K):
    print("logprobs", NAMES[ty], N, V, K, flush=True)
    _, x = on_gpu(rows_of(ty, N, V))
    M = 1 + V % 3
    ids = some_ids(N, V, M, V)
    for scale in (1.0, 1.0 / 0.7):
        check_logprobs(logprobs(lib, x, ty, scale, ids, K), x, scale, ids, K)


@pytest.mark.parametrize("ty,N,V,K,pad", [
    (F32, 1030, 1000, 8, 0), (BF16, 1027, 2048, 48, 0), (F16, 1025, 1999, 3, 1),         # a wave a row, in registers
    (F32, 1026, 2048, 40, 0), (F32, 1024, 1500, 1, 3),                                    # eight vectors a lane
    (F32, 2003, 4000, 20, 0), (BF16, 1601, 6001, 48, 1), (F16, 2048, 8100, 10, 4),        # a wave a row, read again
    (F32, 1030, 1000, 49, 0), (BF16, 600, 4096, 128, 0),                                  # four waves
    (F32, 5, 40000, 128, 1), (F16, 40, 66000, 30, 0), (BF16, 300, 80000, 7, 1),           # rows in segments
    (F32, 1, 400000, 128, 0), (BF16, 2, 1 << 20, 100, 0)])
def test_logprobs_every_launch(lib, ty, N, V, K, pad):
    """The sizes at which the launches change: one wave a row or four, parts in
    registers or read again, rows cut into segments."""
    print("launch", NAMES[ty], N, V, K, pad, flush=True)
    _, x = on_gpu(rows_of(ty, N, V, V + pad, 1 if pad else 0))
    x[0] = 0.5                                           # every value the same
    x[N // 2, : V // 2] = 7.0
    x[N - 1, V // 3:] = -math.inf
    ids = some_ids(N, V, 2, V)
    check_logprobs(logprobs(lib, x, ty, 0.9, ids, K), x, 0.9, ids, K)


@pytest.mark.parametrize("ty,N,V,K,pad", [
    (F32, 2560, 2048, 40, 0), (BF16, 2559, 2048, 40, 0), (F16, 2050, 2047, 32, 1), (BF16, 2047, 1000, 32, 0),     # in registers
    (F32, 4100, 2048, 41, 0), (F16, 1280, 999, 20, 3),
    (F32, 3840, 2800, 20, 0), (BF16, 3839, 4801, 20, 1), (F16, 6150, 2100, 32, 0), (F32, 2048, 4096, 10, 0)])     # read again
def test_logprobs_launches_by_alternatives(lib, ty, N, V, K, pad):
    """Where the number of alternatives decides between one wave a row and four."""
    print("launch", NAMES[ty], N, V, K, pad, flush=True)
    _, x = on_gpu(rows_of(ty, N, V, V + pad, 1 if pad else 0))
    x[0] = 0.5
    x[N // 2, : V // 2] = 7.0
    x[N - 1, V // 3:] = -math.inf
    ids = some_ids(N, V, 2, V)
    check_logprobs(logprobs(lib, x, ty, 0.9, ids, K), x, 0.9, ids, K)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("N,V,ld,off", [(3, 1000, 1003, 1), (2, 2048, 2051, 3), (5, 333, 340, 7), (2, 40001, 40010, 5),
                                        (300, 777, 900, 2)])
def test_logprobs_any_alignment_and_stride(lib, ty, N, V, ld, off):
    """Rows that start at every element offset; NaN lies between the rows."""
    print("alignment", NAMES[ty], N, V, ld, off, flush=True)
    _, x = on_gpu(rows_of(ty, N, V, ld, off))
    ids = some_ids(N, V, 2, V)
    check_logprobs(logprobs(lib, x, ty, 1.0, ids, 10), x, 1.0, ids, 10)


def test_logprobs_optional_outputs(lib):
    """No given tokens, no alternatives, no statistics asked for: what is
    written is the same."""
    t = _t()
    for N, V in ((3, 300), (1, 70000), (300, 3000)):
        _, x = on_gpu(rows_of(F32, N, V))
        ids = some_ids(N, V, 1, 3)
        full = logprobs(lib, x, F32, 1.0, ids, 9)
        nb = lib.tlg_logprobs_ws_bytes(F32, N, V, 0)
        ws = t.empty(nb + 16, dtype=t.uint8, device="cuda")
        lg = t.full((N, 1), float("nan"), device="cuda")
        lib.logprobs(x.data_ptr(), F32, V, N, V, 1.0, ids.data_ptr(), 1, lg.data_ptr(), None, None, 0, None, None,
                     ws.data_ptr(), nb, stream())
        ent = t.full((N,), float("nan"), device="cuda")
        lib.logprobs(x.data_ptr(), F32, V, N, V, 1.0, None, 0, None, None, ent.data_ptr(), 0, None, None,
                     ws.data_ptr(), nb, stream())
        tol = 2 * (rho(V) + 8 * EPS * 20)
        close(f64(lg), f64(full.logp), tol, "logp alone")
        close(f64(ent), f64(full.entropy), tol * math.log(V), "entropy alone")


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("N,V", [(4, 100), (4, 2048), (3, 40000), (260, 5000), (1030, 1000)])
def test_ties_go_to_the_lowest_index(lib, ty, N, V):
    """Rows of equal values, of few different values, of both zeros."""
    t = _t()
    print("ties", NAMES[ty], N, V, flush=True)
    g = t.Generator().manual_seed(5)
    x = t.zeros(N, V)
    x[1] = t.randint(0, 3, (V,), generator=g).float()
    x[2] = t.where(t.rand(V, generator=g) < 0.5, -0.0, 0.0)
    if N > 3:
        x[3] = -t.randint(0, V // 50 + 1, (V,), generator=g).float() / 16
    x = x.to(dtype(ty)).cuda()
    for K in (1, 7, 64, 128):
        check_logprobs(logprobs(lib, x, ty, 1.0, None, K), x, 1.0, None, K)


@pytest.mark.parametrize("ty", [F32, BF16])
@pytest.mark.parametrize("step", [1, 4, 8, 64 * 4, 64 * 8, 256 * 4, 256 * 8, 1024 * 4, 1024 * 8])
def test_alternatives_that_lie_together(lib, ty, step):
    """The largest values all in one column of the row's vectors (the same
    thread's, whatever the kernel's width), ascending and descending, and rows
    in sorted order: far more candidates than a random row has."""
    t = _t()
    print("together", NAMES[ty], step, flush=True)
    for V in (2048, 60000):
        g = t.Generator().manual_seed(step)
        x = t.randn(4, V, generator=g)
        at = t.arange(3 if V > 3 else 0, V, step)[:700]
        x[0, at] = 20.0 + t.arange(len(at)) / 16
        x[1, at] = 90.0 - t.arange(len(at)) / 16
        x[2] = t.arange(V) / 4096
        x[3] = -t.arange(V) / 4096
        x = x.to(dtype(ty)).cuda()
        for K in (5, 128):
            check_logprobs(logprobs(lib, x, ty, 1.0, None, K), x, 1.0, None, K)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("V", [5, 300, 2048, 33001])
@pytest.mark.parametrize("N", [8, 520])
def test_masked_rows_infinities_and_nan(lib, ty, V, N):
    """Rows that the mask leaves nothing or little of, the type's lowest value
    as a mask, NaN and infinities, in the first eight of N rows."""
    t = _t()
    if N * V > 1 << 23:
        N = 200
    print("masked", NAMES[ty], N, V, flush=True)
    lo = t.finfo(dtype(ty)).min
    g = t.Generator().manual_seed(V)
    x = 2 * t.randn(N, V, generator=g)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, V - 1] = 3.0
    x[2] = lo
    x[3, : V - 2] = lo
    x[4, V // 2] = math.nan
    x[5, V // 3] = math.inf
    x[6, t.rand(V, generator=g) < 0.9] = -math.inf
    x[7] = -math.inf
    x[7, 0], x[7, V // 2] = lo, -math.inf
    x = x.to(dtype(ty)).cuda()
    ids = some_ids(N, V, 3, V)
    ids[2, 1] = V + 3
    ids[0, 0], ids[0, 1] = 0, -1
    check_logprobs(logprobs(lib, x, ty, 1.0, ids, 12), x, 1.0, ids, 12)


@pytest.mark.parametrize("N,V", [(9, 300), (9, 9000), (3, 50000), (1100, 2048), (9, 2048)])
def test_large_finite_masks_and_values(lib, N, V):
    """Masks of -1e5 .. -1e38 over parts of a row (whole lanes, waves and
    segments of it), over all of it, and logits as large as that."""
    t = _t()
    print("large", N, V, flush=True)
    g = t.Generator().manual_seed(V)
    base = 2 * t.randn(N, V, generator=g)
    for far in (1e5, 1e6, 1e7, 1e9, 1e10, 1e20, 3e38):
        x = base.clone()
        x[0] = -far
        x[1, 7:] = -far
        x[2, : V - 1] = -far
        if N > 3:
            x[3, t.rand(V, generator=g) < 0.9] = -far
            x[4] = far
            x[5, V // 2] = far
            x[6, V // 3] = -far
            x[7, :: 2] = -far
            x[8, V // 4: V // 2] = -far
        for ty in (F32, BF16):
            y = x.to(dtype(ty)).cuda()
            ids = some_ids(N, V, 2, 1)
            check_logprobs(logprobs(lib, y, ty, 1.0, ids, 5), y, 1.0, ids, 5)
            tgt = ids[:, 1].contiguous()
            _, d = like_rows(y, ty)
            o = distill(lib, y, ty, None, None, False, 1.0, 1.0, tgt, 1.0, d)
            rows, grad = ref_distill(f64(y), np.zeros((N, 0), int), np.zeros((N, 0)), False, 1.0, 1.0, tgt.cpu().numpy(), 1.0)
            # differences of values this large are exact or off by half a step of theirs
            close(f64(o.rows), rows, 3 * rho(V) + 8 * EPS * (60 + np.abs(rows)), "rows")
            close(f64(d), grad, (half_step(ty) * 1.01 + 8 * EPS) * np.abs(grad) + 2 * rho(V) + 200 * EPS, "dlogits")


@pytest.mark.parametrize("ty", [F32, BF16])
@pytest.mark.parametrize("N,V", [(3, 40), (5, 300), (2, 70001), (1030, 1000)])
def test_differences_beyond_the_type(lib, ty, N, V):
    """Logits farther apart than fp32 reaches: scaled, their log probabilities
    and a weighted loss are ordinary numbers."""
    t = _t()
    print("beyond", NAMES[ty], N, V, flush=True)
    _, x = on_gpu(rows_of(ty, N, V))
    x[0, 3], x[0, 7:20], x[0, 30] = 3e38, -3e38, -math.inf
    x[1, V - 1], x[1, 5] = 2e38, -2.5e38
    ids = some_ids(N, V, 3, 1, none=False)
    ids[:2, 0], ids[:2, 1], ids[0, 2] = 7, 5, 30
    K = 40 if N > 1000 else 128
    for scale in (float(np.float32(1e-30)), 0.25):
        check_logprobs(logprobs(lib, x, ty, scale, ids, K), x, scale, ids, K)
    X = f64(x)
    tids = t.tensor([[3, 7, 9]], dtype=t.int32, device="cuda").repeat(N, 1)
    tids[1, 1] = 5
    tl = t.full((N, 3), math.log(0.25), device="cuda")
    tgt = tids[:, 1].contiguous()
    for tail in (False, True):
        o = distill(lib, x, ty, tids, tl, tail, 1.0, 1e-6, tgt, 1e-6, None)
        # q is 1/4 each, and 1/4 remains, or 1/3 each; log p_r in the logarithms' domain (e^-3e38 is 0)
        lp, I = ref_logp(X, 1.0)[0], tids.cpu().numpy().astype(np.int64)
        q = math.exp(float(tl[0, 0])) if tail else 1.0 / 3.0
        qr = 1.0 - 3.0 * q if tail else 0.0
        rest = lp.copy()
        np.put_along_axis(rest, I, -np.inf, 1)
        top = rest.max(1)
        with np.errstate(divide="ignore"):
            lpr = top + np.log(np.exp(rest - top[:, None]).sum(1))
        kl = (q * (math.log(q) - np.take_along_axis(lp, I, 1))).sum(1)
        if tail:
            kl += qr * (math.log(qr) - lpr)
        rows = 1e-6 * (kl - lp[np.arange(N), I[:, 1]])
        # weights as rounded to fp32, the remainder's parts and the last rounding: a half step
        # each; ordinary rows as elsewhere
        close(f64(o.rows), rows, 6 * EPS * np.abs(rows) + 1e-6 * (6 * rho(V) + 12 * EPS * 60), "rows")


def test_extreme_temperatures(lib):
    """Almost greedy and almost uniform distributions."""
    _, x = on_gpu(rows_of(F32, 5, 3000))
    ids = some_ids(5, 3000, 2, 1)
    for scale in (1e-4, 50.0, 2000.0):
        check_logprobs(logprobs(lib, x, F32, scale, ids, 6), x, scale, ids, 6)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("N,V", [(3, 300), (2, 70001), (1030, 1000), (41, 40003)])
def test_smallest_and_largest_temperatures(lib, ty, N, V):
    """Scales and temperatures at both ends of their range, over masked tokens
    and logits whose scaled values pass fp32."""
    t = _t()
    print("temperatures", NAMES[ty], N, V, flush=True)
    lo, hi = float(np.float32(1e-30)), float(np.float32(1e30))
    _, x = on_gpu(rows_of(ty, N, V))
    x[0, ::3] = -math.inf
    ids = some_ids(N, V, 2, 1)
    for scale in (lo, hi):
        check_logprobs(logprobs(lib, x, ty, scale, ids, 20), x, scale, ids, 20)
    if ty != F16:
        y = x.clone()
        y[1, 11], y[1, 40:50], y[0, 20:] = 3e38, -3e38, -3e38
        check_logprobs(logprobs(lib, y, ty, hi, None, 0), y, hi, None, 0)
    tids, tl = teacher(x, 8, 1.0)
    x[1] = 0.25
    X, I, q = f64(x), tids.cpu().numpy().astype(np.int64), np.exp(f64(tl))
    for tau in (lo, hi):
        p = np.exp(ref_logp(X, 1.0 / tau)[0])
        Xo = X.copy()
        np.put_along_axis(Xo, I, -np.inf, 1)
        po = np.exp(ref_logp(Xo, 1.0 / tau)[0])          # among the tokens the teacher does not name
        for tail in (False, True):
            _, d = like_rows(x, ty)
            scale = float(np.float32(1.0 / tau))         # so that the gradient is an ordinary number
            distill(lib, x, ty, tids, tl, tail, tau, 1.0, None, 0.0, d, scale)
            Q = q.sum(1, keepdims=True)
            want = p.copy()
            np.put_along_axis(want, I, np.take_along_axis(p, I, 1) - (q if tail else q / Q), 1)
            if tail:
                want -= (1.0 - Q) * po
            # p and po: sums and exponentials; q in 64 bits; a few roundings of the factors
            # tau, scale and their product; the output's half step
            bar = (p + tail * po) * (4 * rho(V) + 40 * EPS) + (half_step(ty) * 1.01 + 20 * EPS) * np.abs(want) + 8 * EPS
            close(f64(d), want, bar, ("dlogits", tau, tail))


# ---------------------------------------------------------------- gradient --
def grad_tol(ty, X, scale, want, c0, c1, H, factor):
    """|d p| <= p eps (4 |z'| + 2 |log S| + 8) for the recomputed probabilities,
    its products with the coefficients, and the output's rounding."""
    lp, _, ls, _ = ref_logp(X, scale)
    with np.errstate(all="ignore"):
        p = np.where(np.isfinite(lp), np.exp(lp), 0.0)
        a = np.where(np.isfinite(lp), np.abs(lp), 0.0)
        l = np.abs(np.where(np.isfinite(ls), ls, 0.0))[:, None]
        h = np.abs(H)[:, None]
        relp = EPS * (4 * (a + l) + 2 * l + 8)
        t = p * (np.abs(c0)[:, None] * (relp + 80 * EPS) +
                 np.abs(c1)[:, None] * (relp * (a + h) + 8 * EPS * (a + l + h + 1)))
    return factor * t * 1.01 + (half_step(ty) * 1.01 + 70 * EPS) * np.abs(want) + tiny(ty)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("N,V,M,pad,off", [(1, 1, 1, 0, 0), (3, 2, 2, 1, 1), (5, 65, 64, 0, 0), (4, 1000, 3, 3, 1),
                                           (130, 2048, 1, 0, 0), (7, 2049, 5, 8, 3), (2, 40001, 4, 9, 5),
                                           (1, 131072, 1, 0, 0)])
def test_logprobs_bwd(lib, ty, N, V, M, pad, off):
    t = _t()
    print("logprobs_bwd", NAMES[ty], N, V, M, pad, off, flush=True)
    _, x = on_gpu(rows_of(ty, N, V, V + pad, off))
    ids = some_ids(N, V, M, V)
    g = t.Generator().manual_seed(V + 1)
    dlogp, dlse, dent = (t.randn(*s, generator=g).cuda() for s in ((N, M), (N,), (N,)))
    scale = 1.0 / 1.3
    X = f64(x)
    _, m, ls, H = ref_logp(X, scale)
    lse2 = t.tensor(np.stack([m, ls], 1), dtype=t.float32, device="cuda")
    ent = t.tensor(H, dtype=t.float32, device="cuda")
    I, dl = ids.cpu().numpy(), f64(dlogp)
    for use_lse, use_ent in ((True, True), (False, False), (False, True)):
        a, b = (f64(dlse) if use_lse else np.zeros(N)), (f64(dent) if use_ent else np.zeros(N))
        buf, d = like_rows(x, ty)
        logprobs_bwd(lib, x, ty, scale, ids, lse2, ent, dlogp, dlse if use_lse else None, dent if use_ent else None, d)
        want = ref_bwd(X, scale, I, dl, a, b)
        c0 = np.abs(np.where(I >= 0, dl, 0.0)).sum(1) + np.abs(a)
        tol = grad_tol(ty, X, scale, want, c0, b, H, scale)
        # the given tokens' own terms cancel against p's
        for n in range(N):
            for j, i in enumerate(I[n]):
                if i >= 0:
                    tol[n, i] += scale * abs(dl[n, j]) * (M + 4) * EPS
        close(f64(d), want, tol, "dlogits")
        guard = buf.clone()
        t.as_strided(guard, tuple(d.shape), (d.stride(0), 1), d.storage_offset()).fill_(float("nan"))
        assert bool(t.isnan(guard).all()), "wrote outside its rows"


def test_logprobs_bwd_in_place_and_repeated_ids(lib):
    t = _t()
    for ty in (F32, F16, BF16):
        for N, V in ((70, 2051), (2, 50000)):
            buf, x = on_gpu(rows_of(ty, N, V, V + 5, 1))
            ids = some_ids(N, V, 6, 9)
            ids[:, 3] = ids[:, 1]
            f = logprobs(lib, x, ty, 1.0, ids, 0)
            dlogp = t.randn(N, 6, device="cuda")
            dent = t.randn(N, device="cuda")
            _, d = like_rows(x, ty)
            logprobs_bwd(lib, x, ty, 1.0, ids, f.lse2, f.entropy, dlogp, None, dent, d)
            merged = ids.clone()
            merged[:, 3] = -1
            dm = dlogp.clone()
            dm[:, 1] += dm[:, 3]
            _, d2 = like_rows(x, ty)
            logprobs_bwd(lib, x, ty, 1.0, merged, f.lse2, f.entropy, dm, None, dent, d2)
            # the same sum in another order: a few roundings of the coefficients
            lim = 16 * EPS * float(dlogp.abs().sum(1).max()) + half_step(ty) * 2.1 * float(d.abs().max())
            assert float((d.double() - d2.double()).abs().max()) <= lim
            logprobs_bwd(lib, x, ty, 1.0, ids, f.lse2, f.entropy, dlogp, None, dent, x)      # in place
            assert t.equal(x, d)


def test_logprobs_bwd_special_rows(lib):
    """Masked rows give 0, padded rows 0 over any logits, NaN rows and token
    ids past the vocabulary NaN."""
    t = _t()
    for N, V in ((8, 300), (8, 70001), (600, 2048)):
        _, x = on_gpu(rows_of(F32, N, V))
        x[0] = -math.inf
        x[1, 5] = math.nan
        x[2, 7] = math.nan
        x[3, : V // 2] = -math.inf
        ids = some_ids(N, V, 2, 4, none=False)
        ids[0] = t.tensor([0, 3])
        ids[2] = -1
        ids[4, 1] = V
        x[7] = -math.inf
        ids[7, 0] = V                                    # a bad id in a row that is masked
        f = logprobs(lib, x, F32, 1.0, ids, 0)
        dlogp, dent = t.randn(N, 2, device="cuda"), t.randn(N, device="cuda")
        dent[2] = 0.0
        _, d = like_rows(x, F32)
        logprobs_bwd(lib, x, F32, 1.0, ids, f.lse2, f.entropy, dlogp, None, dent, d)
        assert bool((d[0] == 0).all()) and bool((d[2] == 0).all())
        assert bool(t.isnan(d[1]).all()) and bool(t.isnan(d[4]).all()) and bool(t.isnan(d[7]).all())
        part = ids[3, 0] >= V // 2
        assert bool((d[3, : V // 2][t.arange(V // 2, device="cuda") != ids[3, 0]][:100].isfinite()).all()) or part
        assert bool(d[5:7].isfinite().all()) and bool(d[8:].isfinite().all())


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("N,V", [(8, 300), (8, 70001), (600, 2048)])
@pytest.mark.parametrize("how", ["pair", "lse", "same token"])
def test_logprobs_bwd_coefficients_that_cancel(lib, ty, N, V, how):
    """Coefficients that cancel in their sum are no padding: the gradient of a
    finite row is theirs at the given tokens alone, that of a NaN or +inf row NaN."""
    t = _t()
    print("cancel", NAMES[ty], N, V, how, flush=True)
    _, x = on_gpu(rows_of(ty, N, V))
    x[1, 5], x[2, 7], x[4] = math.nan, math.inf, math.nan
    x[3] = -math.inf
    x[5, 9] = math.nan
    ids = t.tensor([[11, V - 2]], dtype=t.int32, device="cuda").repeat(N, 1)
    dlogp = t.tensor([[0.75, -0.75]], device="cuda").repeat(N, 1)
    dlse = None
    if how == "lse":
        dlogp[:, 1] = 0.5
        dlse = dlogp.sum(1)                              # 1.25: exact
        dlse[4] = 0.0
    elif how == "same token":
        ids[:, 1] = ids[:, 0]
    ids[4] = -1                                          # a padded row over NaN
    dlogp[5] = 0.0                                       # one whose coefficients are all 0
    if dlse is not None:
        dlse[5] = 0.0
    f = logprobs(lib, x, ty, 1.0, ids, 0)
    _, d = like_rows(x, ty)
    logprobs_bwd(lib, x, ty, 1.0, ids, f.lse2, None, dlogp, dlse, None, d)
    assert bool(t.isnan(d[1]).all()) and bool(t.isnan(d[2]).all()), "a NaN row"
    assert not bool(d[3:6].any()), "a masked row, a padded one and one without coefficients"
    want = t.zeros(N, V, device="cuda")
    want.scatter_add_(1, ids.clamp(min=0).long(), dlogp)
    good = [0] + list(range(6, N))
    assert t.equal(d[good].float(), want[good])          # 0.75 and 0.5 are exact in every type


def test_logprobs_gradient_against_differences(lib):
    """Directional central differences of the kernel's own forward."""
    t = _t()
    N, V, h = 6, 1500, 1.0 / 64
    _, x = on_gpu(rows_of(F32, N, V))
    ids = some_ids(N, V, 2, 11, none=False)
    dlogp, dlse, dent = t.randn(N, 2, device="cuda"), t.randn(N, device="cuda"), t.randn(N, device="cuda")

    def value(y):
        o = logprobs(lib, y, F32, 0.8, ids, 0)
        lse = 0.8 * o.lse2[:, 0].double() + o.lse2[:, 1].double()
        return (dlogp.double() * o.logp.double()).sum(1) + dlse.double() * lse + dent.double() * o.entropy.double()
    f = logprobs(lib, x, F32, 0.8, ids, 0)
    _, d = like_rows(x, F32)
    logprobs_bwd(lib, x, F32, 0.8, ids, f.lse2, f.entropy, dlogp, dlse, dent, d)
    v = (t.randn(N, V, device="cuda") * 4).round().clamp(-8, 8) / 4          # x +- h v in few bits
    num = (value(x + h * v) - value(x - h * v)) / (2 * h)
    ana = (d.double() * v.double()).sum(1)
    # third derivatives of these sums are at most a few times |v|^3 (cumulants of
    # a variable in [-2, 2], entropy's with a factor log V); fp32 values / h
    c = (dlogp.abs().sum(1) + dlse.abs() + dent.abs() * math.log(V)).double() + 1
    bar = c * (h * h / 6 * 8 * 8 + 4 * (rho(V) * 2 * math.log(V) + 60 * EPS) / h)
    assert bool(((num - ana).abs() <= bar).all()), (num, ana, bar)
    assert float((ana.abs() / bar).max()) > 3, "differences that could not fail"


# -------------------------------------------------------------- distillation --
def teacher(x, K, tau, seed=1, noise=0.5):
    t = _t()
    g = t.Generator().manual_seed(seed)
    y = (x.float().cpu().nan_to_num(0.0, 0.0, -30.0) + noise * t.randn(tuple(x.shape), generator=g)).double() / tau
    lp = t.log_softmax(y, 1)
    K1 = min(K, x.shape[1])
    v, i = t.topk(lp, K1, dim=1)
    ids, tl = t.full((x.shape[0], K), -1, dtype=t.int32), t.zeros(x.shape[0], K)
    ids[:, :K1], tl[:, :K1] = i.int(), v.float()
    return ids.cuda(), tl.cuda()


def check_distill(o, d, ty, x, ids, tl, tail, tau, w_kd, tgt, w_ce, scale):
    X = f64(x)
    N, V = X.shape
    I = np.zeros((N, 0), np.int64) if ids is None else ids.cpu().numpy()
    T = np.zeros((N, 0)) if tl is None else f64(tl)
    G = None if tgt is None else tgt.cpu().numpy()
    rows, grad = ref_distill(X, I, T, tail, tau, w_kd, G, w_ce)
    lp, _, ls, _ = ref_logp(X, 1.0 / tau)
    lp1, _, ls1, _ = ref_logp(X, 1.0)
    # rows: log probabilities off by tol_lp each, weighted by sum q = 1 (and the
    # remainder's log p_r by rho twice); teacher terms are in 64 bits
    fin = np.isfinite(rows)
    a = np.where(np.isfinite(lp), np.abs(lp), 0.0).max(1) if V < 100000 else np.full(N, 60.0)
    a1 = np.where(np.isfinite(lp1), np.abs(lp1), 0.0).max(1) if V < 100000 else np.full(N, 60.0)
    tol = w_kd * tau * tau * (3 * rho(V) + 6 * EPS * (a + np.abs(ls))) + \
        w_ce * (2 * rho(V) + 6 * EPS * (a1 + np.abs(ls1))) + 2 * EPS * np.abs(np.where(fin, rows, 0.0))
    close(f64(o.rows), rows, tol, "rows")
    if fin.all():
        close(f64(o.loss), [rows.mean()], tol.mean() + 2 * EPS * abs(rows.mean()), "loss")
    if d is None:
        return
    want = scale * grad
    p, p1 = np.exp(lp), np.exp(lp1)
    # p: exponentials and S; the remainder's Q - q_r / p_r carries 2 rho of its parts
    with np.errstate(all="ignore"):
        z, z1 = np.where(p > 0, np.abs(lp), 0.0), np.where(p1 > 0, np.abs(lp1), 0.0)
        relp = EPS * (4 * (z + np.abs(ls)[:, None]) + 12) + rho(V)
        relp1 = EPS * (4 * (z1 + np.abs(ls1)[:, None]) + 12) + rho(V)
    ratio = np.ones(N)
    if tail:
        for n in range(N):
            S = np.unique(I[n][I[n] >= 0])
            out = np.delete(p[n], S).sum()
            q = sum(math.exp(T[n, list(I[n]).index(s)]) for s in S)
            ratio[n] = 2 + (max(0.0, 1 - q) / out if out > 0 else 0.0)
    q = np.zeros((N, V))
    for n in range(N):
        q[n, I[n][I[n] >= 0]] = 1.0
    bar = abs(scale) * (w_kd * tau * (p * ratio[:, None] * (relp + 3 * rho(V)) + q * 4 * EPS) +
                        w_ce * (p1 * relp1 + 4 * EPS * (p1 > 1e-30)) * (0 if G is None else 1))
    bar = bar + (half_step(ty) * 1.01 + 8 * EPS) * np.abs(want) + tiny(ty)
    close(f64(d), want, bar, "dlogits")


KD = [  # N, V, K, tail, tau, w_kd, w_ce, pad, off
    (1, 2, 1, False, 1.0, 1.0, 0.0, 0, 0), (3, 5, 4, True, 1.0, 1.0, 0.5, 2, 1), (2, 7, 9, True, 2.0, 0.5, 0.5, 0, 0),
    (5, 64, 64, False, 1.0, 1.0, 1.0, 0, 0), (4, 257, 20, True, 1.5, 1.0, 0.0, 1, 3), (3, 1000, 128, True, 1.0, 1.0, 0.3, 3, 1),
    (70, 2048, 8, False, 2.0, 0.7, 0.3, 0, 0), (300, 2048, 32, True, 1.0, 1.0, 0.5, 0, 0), (9, 2051, 16, False, 0.7, 1.0, 0.0, 6, 5),
    (2, 8192, 50, True, 1.0, 1.0, 0.0, 0, 0), (3, 16385, 64, False, 1.0, 1.0, 1.0, 3, 2), (2, 40001, 50, True, 1.0, 1.0, 0.5, 9, 5),
    (1, 131072, 100, True, 1.0, 1.0, 0.0, 0, 0), (257, 5003, 12, True, 2.0, 1.0, 0.5, 0, 0), (2, 70000, 0, False, 1.0, 1.0, 1.0, 0, 0)]


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("N,V,K,tail,tau,w_kd,w_ce,pad,off", KD)
def test_distill(lib, ty, N, V, K, tail, tau, w_kd, w_ce, pad, off):
    t = _t()
    print("distill", NAMES[ty], N, V, K, tail, flush=True)
    _, x = on_gpu(rows_of(ty, N, V, V + pad, off))
    ids, tl = teacher(x, K, tau) if K else (None, None)
    tgt = t.randint(0, V, (N,), generator=t.Generator().manual_seed(2), dtype=t.int32).cuda()
    if K and N > 1:
        tgt[1] = ids[1, 0]                     # a target that the teacher names too
    if N > 2:
        tgt[2] = -1
    if K and N > 4:
        ids[3] = -1
        ids[4], tgt[4] = -1, -1                # a padded row
    scale = 1.0 / N
    buf, d = like_rows(x, ty)
    o = distill(lib, x, ty, ids, tl, tail, tau, w_kd, tgt if w_ce else None, w_ce, d, scale)
    check_distill(o, d, ty, x, ids, tl, tail, tau, w_kd, tgt if w_ce else None, w_ce, scale)
    guard = buf.clone()
    t.as_strided(guard, tuple(d.shape), (d.stride(0), 1), d.storage_offset()).fill_(float("nan"))
    assert bool(t.isnan(guard).all()), "wrote outside its rows"
    # the loss alone, and in place
    o2 = distill(lib, x, ty, ids, tl, tail, tau, w_kd, tgt if w_ce else None, w_ce, None, scale)
    assert t.equal(o2.rows, o.rows) and t.equal(o2.loss, o.loss)
    o3 = distill(lib, x, ty, ids, tl, tail, tau, w_kd, tgt if w_ce else None, w_ce, x, scale)
    assert t.equal(o3.rows, o.rows) and t.equal(x, d)


@pytest.mark.parametrize("ty,N,V,K,tail,tau,pad", [
    (F32, 2050, 1000, 8, True, 2.0, 0), (BF16, 2049, 2048, 70, False, 1.0, 0), (F16, 2051, 1500, 5, True, 1.0, 3),
    (F32, 2048, 2048, 32, True, 1.0, 0), (F32, 2050, 2000, 32, False, 2.0, 1),
    (F32, 20, 3000, 20, True, 2.0, 0), (BF16, 20, 8000, 20, True, 1.0, 1),
    (F32, 20, 8000, 128, True, 1.0, 0), (F16, 20, 16000, 20, False, 2.0, 1),
    (F32, 20, 16000, 20, True, 2.0, 1), (BF16, 20, 30000, 65, True, 1.0, 0),
    (F32, 130, 32000, 20, True, 1.0, 0), (F32, 200, 50000, 20, True, 1.0, 1), (F32, 260, 40000, 9, False, 1.0, 0),
    (F32, 140, 33000, 20, True, 2.0, 0), (BF16, 135, 66000, 20, True, 1.0, 1), (F16, 200, 40000, 20, True, 2.0, 0),
    (F32, 3, 50000, 128, True, 2.0, 1), (BF16, 10, 131000, 64, True, 1.0, 0), (F32, 1, 1 << 20, 100, True, 1.0, 0)])
def test_distill_every_launch(lib, ty, N, V, K, tail, tau, pad):
    """The sizes at which the launches change: one to sixteen waves a row, rows
    in registers or read twice, rows cut into segments."""
    t = _t()
    print("distill launch", NAMES[ty], N, V, K, tail, tau, flush=True)
    _, x = on_gpu(rows_of(ty, N, V, V + pad, 1 if pad else 0))
    ids, tl = teacher(x, K, tau)
    ids[N // 2, K // 2] = ids[N // 2, 0]                 # a repeated id
    tgt = t.randint(0, V, (N,), generator=t.Generator().manual_seed(2), dtype=t.int32).cuda()
    tgt[0] = ids[0, K - 1]
    buf, d = like_rows(x, ty)
    o = distill(lib, x, ty, ids, tl, tail, tau, 1.0, tgt, 0.5, d, 0.25)
    pick = sorted(set(list(range(0, N, max(1, N // 60))) + [N // 2, N - 1]))
    o.rows, dd = o.rows[pick], d[pick]
    whole = o.loss.clone()
    o.loss = o.rows.double().mean().float().reshape(1)
    check_distill(o, dd, ty, x[pick], ids[pick], tl[pick], tail, tau, 1.0, tgt[pick], 0.5, 0.25)
    o2 = distill(lib, x, ty, ids, tl, tail, tau, 1.0, tgt, 0.5, x, 0.25)          # in place
    assert t.equal(x, d) and t.equal(o2.loss, whole)
    assert abs(float(whole) - float(o2.rows.double().mean())) <= 2 * EPS * abs(float(whole))
    t.as_strided(buf, tuple(d.shape), (d.stride(0), 1), d.storage_offset()).fill_(float("nan"))
    assert bool(t.isnan(buf).all()), "wrote outside its rows"


@pytest.mark.parametrize("ty,N,V,tau,pad", [
    (F32, 20, 16388, 2.0, 0), (F32, 33, 24577, 1.0, 3), (F32, 35, 32771, 1.0, 0), (F32, 45, 41001, 2.0, 1),
    (F32, 60, 57350, 1.0, 0), (F32, 130, 131077, 2.0, 0), (F32, 260, 262144, 1.0, 0),
    (F16, 20, 20000, 2.0, 0), (BF16, 20, 32769, 1.0, 7), (F16, 21, 33001, 2.0, 1), (BF16, 22, 41001, 2.0, 0),
    (BF16, 25, 49153, 1.0, 0), (F16, 40, 65530, 1.0, 5), (BF16, 44, 90001, 1.0, 0), (F16, 70, 131072, 1.0, 0),
    (BF16, 140, 262147, 1.0, 1)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_rows_read_twice(lib, ty, N, V, tau, pad, tail):
    """Every number of rounds: all of a row's kept in registers, the first ones in
    LDS, the rest read again; the last round full, partly full or one vector."""
    t = _t()
    print("distill twice", NAMES[ty], N, V, tau, pad, tail, flush=True)
    _, x = on_gpu(rows_of(ty, N, V, V + pad, 1 if pad else 0))
    ids, tl = teacher(x, 40, tau)
    ids[:, 1] = V - 1                                    # an id in each row's last round
    ids[:, 2] = t.arange(N, dtype=t.int32, device="cuda") * 257 % V
    tgt = t.randint(0, V, (N,), generator=t.Generator().manual_seed(2), dtype=t.int32).cuda()
    buf, d = like_rows(x, ty)
    o = distill(lib, x, ty, ids, tl, tail, tau, 1.0, tgt, 0.5, d, 0.25)
    pick = [0, 1, N // 2, N - 2, N - 1]
    o.rows, dd = o.rows[pick], d[pick]
    whole = o.loss.clone()
    o.loss = o.rows.double().mean().float().reshape(1)
    check_distill(o, dd, ty, x[pick], ids[pick], tl[pick], tail, tau, 1.0, tgt[pick], 0.5, 0.25)
    o2 = distill(lib, x, ty, ids, tl, tail, tau, 1.0, tgt, 0.5, x, 0.25)          # in place
    assert t.equal(x, d) and t.equal(o2.loss, whole)
    t.as_strided(buf, tuple(d.shape), (d.stride(0), 1), d.storage_offset()).fill_(float("nan"))
    assert bool(t.isnan(buf).all()), "wrote outside its rows"


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,V", [(12, 300), (12, 50003), (530, 2048), (2060, 1200)])
def test_distill_special_rows(lib, tail, N, V):
    """Repeated ids, entries without mass, a support that is all the student
    has, padding over NaN, masked and NaN rows, ids past the vocabulary."""
    t = _t()
    print("distill special", tail, N, V, flush=True)
    _, x = on_gpu(rows_of(F32, N, V, spread=1.5))
    K = 10
    ids, tl = teacher(x, K, 1.0)
    tgt = ids[:, 1].clone()
    ids[0, 4], ids[0, 7] = ids[0, 2], ids[0, 2]      # the first place counts
    tl[1, 3] = -math.inf                             # an entry of the support without mass
    ids[2], tgt[2] = -1, -1                          # a padded row over NaN
    x[2] = math.nan
    x[3] = -math.inf                                 # nothing left
    ids[3], tgt[3] = -1, -1
    x[4, 9] = math.nan
    ids[5, 6] = V
    tl[6] = -math.inf
    x[7, ids[7, 0].long()] = -math.inf               # the student excludes what the teacher wants
    tgt[7] = ids[7, 5]
    tl[8] = tl[8] + 2.0                              # more mass than one
    keep = x[9, ids[9].long()].clone()               # outside the support nothing is left
    x[9] = -math.inf
    x[9, ids[9].long()] = keep
    _, d = like_rows(x, F32)
    o = distill(lib, x, F32, ids, tl, tail, 1.0, 1.0, tgt, 0.5, d)
    rows = f64(o.rows)
    assert rows[2] == 0 and bool((d[2] == 0).all())
    assert rows[3] == 0 and bool((d[3] == 0).all())
    assert np.isnan(rows[4]) and bool(t.isnan(d[4]).all())
    assert np.isnan(rows[5]) and bool(t.isnan(d[5]).all())
    assert rows[7] == math.inf
    good = [0, 1, 6, 7, 8, 9, 10, 11] + list(range(12, N))
    sub = x[good]
    o.rows, dd = o.rows[good], d[good]
    o.loss = o.rows.mean().reshape(1)
    check_distill(o, dd, F32, sub, ids[good], tl[good], tail, 1.0, 1.0, tgt[good], 0.5, 1.0)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,V,w_kd,w_ce", [(9, 300, 1.0, 0.5), (9, 300, 0.0, 0.5), (9, 70000, 1.0, 0.5), (300, 50003, 1.0, 0.0),
                                           (530, 2048, 1.0, 0.5), (2060, 1200, 1.0, 0.5)])
def test_distill_broken_teachers(lib, tail, N, V, w_kd, w_ce):
    """An entry whose log probability is NaN or +inf makes its row's loss and
    gradient NaN, whatever stands beside it; beside a negative id, or at an id's
    second place, it is no entry."""
    t = _t()
    print("broken teacher", tail, N, V, w_kd, w_ce, flush=True)
    _, x = on_gpu(rows_of(F32, N, V))
    K = 70
    ids, tl = teacher(x, K, 2.0)
    ids[3, 4], ids[4, 9], ids[5] = -1, ids[4, 2], -1
    tgt = t.randint(0, V, (N,), generator=t.Generator().manual_seed(2), dtype=t.int32).cuda()
    _, d0 = like_rows(x, F32)
    clean = distill(lib, x, F32, ids, tl, tail, 2.0, w_kd, tgt, w_ce, d0)
    assert bool(clean.rows.isfinite().all()) and bool(d0.isfinite().all())
    tl = tl.clone()
    tl[0] = math.nan                                     # every entry
    tl[1, 3] = math.nan                                  # one of many
    tl[2, 66] = math.inf
    tl[3, 4] = tl[4, 9] = math.nan                       # no entries
    tl[5] = math.nan
    _, d = like_rows(x, F32)
    o = distill(lib, x, F32, ids, tl, tail, 2.0, w_kd, tgt, w_ce, d)
    assert np.isnan(f64(o.rows[:3])).all() and np.isnan(f64(o.loss)).all()
    assert bool(t.isnan(d[:3]).all())
    assert t.equal(o.rows[3:], clean.rows[3:]) and t.equal(d[3:], d0[3:])


def test_distill_largest_vocabulary_in_one_piece(lib):
    """Rows of 2^20 columns that are not cut: the largest bitmap of the ids."""
    t = _t()
    N, V, K = 520, 1 << 20, 64
    x = (2.5 * t.randn(N, V, device="cuda", generator=t.Generator("cuda").manual_seed(1))).bfloat16()
    ids = t.randint(0, V, (N, K), generator=t.Generator().manual_seed(1), dtype=t.int32).cuda()
    tl = (-5.0 - t.rand(N, K, generator=t.Generator().manual_seed(2))).cuda()
    d = t.full((N, V), float("nan"), dtype=t.bfloat16, device="cuda")
    o = distill(lib, x, BF16, ids, tl, True, 1.0, 1.0, None, 0.0, d)
    assert bool(d.isfinite().all())
    pick = [0, 255, N - 1]
    o.rows, o.loss = o.rows[pick], o.rows[pick].mean().reshape(1)
    check_distill(o, d[pick], BF16, x[pick], ids[pick], tl[pick], True, 1.0, 1.0, None, 0.0, 1.0)


def test_distill_targets_past_the_vocabulary(lib):
    t = _t()
    _, x = on_gpu(rows_of(F32, 3, 100))
    tgt = t.tensor([5, 100, 7], dtype=t.int32, device="cuda")
    _, d = like_rows(x, F32)
    o = distill(lib, x, F32, None, None, False, 1.0, 1.0, tgt, 1.0, d)
    assert np.isnan(f64(o.rows)).tolist() == [False, True, False]
    assert bool(t.isnan(d[1]).all()) and bool(d[0].isfinite().all()) and bool(d[2].isfinite().all())


def test_distill_gradient_against_differences(lib):
    t = _t()
    N, V, K, h = 6, 1500, 24, 1.0 / 64
    for tail, tau in ((False, 2.0), (True, 1.0)):
        _, x = on_gpu(rows_of(F32, N, V))
        ids, tl = teacher(x, K, tau, noise=1.5)
        tgt = t.randint(0, V, (N,), dtype=t.int32).cuda()
        _, d = like_rows(x, F32)
        distill(lib, x, F32, ids, tl, tail, tau, 1.0, tgt, 0.5, d)
        v = (t.randn(N, V, device="cuda") * 4).round().clamp(-8, 8) / 4
        up = distill(lib, x + h * v, F32, ids, tl, tail, tau, 1.0, tgt, 0.5, None).rows.double()
        dn = distill(lib, x - h * v, F32, ids, tl, tail, tau, 1.0, tgt, 0.5, None).rows.double()
        num, ana = (up - dn) / (2 * h), (d.double() * v.double()).sum(1)
        # cumulants of a variable in [-2, 2] (third: at most 16), for log S, the
        # remainder's log sum and the CE's log S; fp32 values / h
        bar = h * h / 6 * 16 * (tau * tau * 2 + 1) + 2 * (tau * tau + 1) * (3 * rho(V) + 6 * EPS * 40) / h
        assert float((num - ana).abs().max()) <= bar, (num, ana, bar)
        assert float(ana.abs().max()) > 2 * bar, "differences that could not fail"


def test_cross_entropy_alone_is_xent(lib):
    """K = 0 and w_ce = 1 is tlg_dev_xent without its 1e-12."""
    t = _t()
    N, V = 300, 2048
    _, x = on_gpu(rows_of(F32, N, V))
    tgt = t.randint(0, V, (N,), dtype=t.int32).cuda()
    _, d = like_rows(x, F32)
    o = distill(lib, x, F32, None, None, False, 1.0, 1.0, tgt, 1.0, d, 1.0 / N)
    d2, loss = t.empty_like(d), t.empty(1, device="cuda")
    lib.check(lib.tlg_dev_xent(x.data_ptr(), tgt.data_ptr(), d2.data_ptr(), loss.data_ptr(), 1.0 / N, N, V, stream()),
              "xent")
    assert abs(float(loss) - float(o.loss)) <= (4 * rho(V) + 200 * EPS) * float(loss) + 1e-12 * V * 1e6
    assert float((d - d2).abs().max()) <= (2 * rho(V) + 100 * EPS) / N


@pytest.mark.parametrize("ty,N,V", [(F32, 8192, 2048), (BF16, 2048, 30000), (F32, 1024, 16384)])
def test_log_sums_lean_to_neither_side(lib, ty, N, V):
    """The mean signed error of log S over many rows: each row's is random with
    a deviation below 2e-7 (a few eps), so that the mean's is below 2e-7 /
    sqrt(N); the hardware exponential leans by 3.5e-9 (measured)."""
    t = _t()
    x = (2.5 * t.randn(N, V, device="cuda", generator=t.Generator("cuda").manual_seed(V))).to(dtype(ty))
    o = distill(lib, x, ty, None, None, False, 1.0, 1.0, x.argmax(1).int(), 1.0, None)
    z = x.double()
    err = o.rows.double() - t.log(t.exp(z - z.amax(1, keepdim=True)).sum(1))
    assert abs(float(err.mean())) <= 5 * 2e-7 / math.sqrt(N) + 5e-9, float(err.mean())


@pytest.mark.parametrize("scale", [1.0, 0.9, 1.0 / 0.7])
@pytest.mark.parametrize("ty,N,V", [(F32, 16384, 2048), (BF16, 8192, 30000), (BF16, 2048, 131072), (F32, 256, 1 << 20)])
def test_log_probabilities_lean_to_neither_side(lib, ty, N, V, scale):
    """The mean signed error of log S: its constant, which k_logprobs puts right
    through the entropy sum, and the many small terms of long rows.  Against the fp32 logarithm of the exact S, so that what the
    logarithm's own last bit leans by does not count: a row's error is random
    with a deviation below 6e-7 (two roundings of a number below 16), the mean's
    below that / sqrt(N); the hardware exponential leans by 3.5e-9 (measured).
    One rounding is not random: s + kappa u, where s is a fp32 number and kappa u
    (-5.5e-8 s at scale 1) less than a step of it, 2^-24 s to 2^-23 s: it always
    vanishes or always counts a whole step, depending on s, and is off by half a
    step at most, 2^-24 of s, in one direction.  (Without kappa the mean is off by
    1.7e-7 at scale 0.9; summed an element at a time, by 1.1e-7, 5e-7 and 4e-6 at
    scale 1 / 0.7 in rows of 30000, 131072 and 2^20.)"""
    t = _t()
    x = (2.5 * t.randn(N, V, device="cuda", generator=t.Generator("cuda").manual_seed(V))).to(dtype(ty))
    s = float(np.float32(scale))
    o = logprobs(lib, x, ty, s, None, 0)
    S = t.cat([t.exp((z - z.amax(1, keepdim=True)) * s).sum(1) for z in (c.double() for c in x.split(512))])
    err = o.lse2[:, 1].double() - t.log(S.float()).double()
    print("lean", NAMES[ty], N, V, scale, float(err.mean()), float(err.std()), flush=True)
    assert abs(float(err.mean())) <= 5 * 6e-7 / math.sqrt(N) + 5e-9 + EPS, float(err.mean())


@pytest.mark.parametrize("ty,N,V", [(BF16, 2048, 30000), (BF16, 2048, 131072), (F32, 520, 1 << 20)])
def test_log_sums_of_long_rows_lean_to_neither_side(lib, ty, N, V):
    """As test_log_sums_lean_to_neither_side, for rows whose sums are made of few
    large and very many small terms."""
    t = _t()
    x = (2.5 / 0.7 * t.randn(N, V, device="cuda", generator=t.Generator("cuda").manual_seed(V))).to(dtype(ty))
    o = distill(lib, x, ty, None, None, False, 1.0, 1.0, x.argmax(1).int(), 1.0, None)
    S = t.cat([t.exp(z - z.amax(1, keepdim=True)).sum(1) for z in (c.double() for c in x.split(256))])
    err = o.rows.double() - t.log(S)
    print("lean", NAMES[ty], N, V, float(err.mean()), float(err.std()), flush=True)
    assert abs(float(err.mean())) <= 5 * 2e-7 / math.sqrt(N) + 5e-9, float(err.mean())


def other_rows(N, V, ld, off, ty):
    t = _t()
    b = t.full((off + N * ld + 16,), float("nan"), dtype=dtype(ty), device="cuda")
    return b, t.as_strided(b, (N, V), (ld, 1), off)


def written_elsewhere(run, x, ty, ld, off):
    """run(d) into rows of a layout of their own: the bits that rows like the
    logits' get, and nothing around them."""
    t = _t()
    _, like = like_rows(x, ty)
    run(like)
    buf, d = other_rows(*x.shape, ld, off, ty)
    run(d)
    assert t.equal(d, like) and bool(like.isfinite().all())
    d.fill_(float("nan"))
    assert bool(t.isnan(buf).all()), "wrote outside its rows"


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("N,V,pad,off,ld,doff", [
    (5, 333, 3, 1, 333, 0), (5, 333, 0, 0, 341, 3), (300, 2049, 7, 2, 2049, 5), (1030, 1001, 0, 0, 1008, 8), (2100, 1001, 7, 1, 1003, 0),
    (9, 8191, 1, 3, 8192, 0), (9, 16001, 0, 1, 16004, 4), (45, 40001, 6, 0, 40001, 1), (2, 131070, 2, 0, 131071, 3)])
def test_gradients_of_another_layout(lib, ty, N, V, pad, off, ld, doff):
    """Padded logits with a dense gradient and the reverse, in every launch: rows
    in registers, read twice, cut."""
    t = _t()
    print("layout", NAMES[ty], N, V, pad, off, ld, doff, flush=True)
    _, x = on_gpu(rows_of(ty, N, V, V + pad, off))
    ids = some_ids(N, V, 2, V)
    f = logprobs(lib, x, ty, 1.0, ids, 0)
    dlogp, dent = t.randn(N, 2, device="cuda"), t.randn(N, device="cuda")
    written_elsewhere(lambda d: logprobs_bwd(lib, x, ty, 1.0, ids, f.lse2, f.entropy, dlogp, None, dent, d), x, ty, ld, doff)
    tids, tl = teacher(x, 8, 2.0)
    tgt = ids[:, 1].contiguous()
    for tail, w_ce in ((False, 0.0), (True, 0.5)):
        written_elsewhere(lambda d: distill(lib, x, ty, tids, tl, tail, 2.0, 1.0, tgt, w_ce, d), x, ty, ld, doff)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
def test_gradients_at_every_pair_of_alignments(lib, ty):
    t = _t()
    VE, N, V = 4 if ty == F32 else 8, 3, 61
    for off in range(VE):
        _, x = on_gpu(rows_of(ty, N, V, V + 3, off))
        ids = some_ids(N, V, 2, V)
        f = logprobs(lib, x, ty, 1.0, ids, 0)
        dlogp = t.randn(N, 2, device="cuda")
        tids, tl = teacher(x, 5, 1.0)
        for doff in range(VE):
            written_elsewhere(lambda d: logprobs_bwd(lib, x, ty, 1.0, ids, f.lse2, None, dlogp, None, None, d), x, ty, V + 5, doff)
            written_elsewhere(lambda d: distill(lib, x, ty, tids, tl, True, 1.0, 1.0, None, 0.0, d), x, ty, V + 5, doff)


@pytest.mark.parametrize("ty", [F32, F16, BF16])
def test_logprobs_bwd_without_given_tokens(lib, ty):
    """M = 0: the gradient of the entropy or of the log-sum-exp alone."""
    t = _t()
    for N, V in ((5, 300), (2, 40001), (130, 2048)):
        print("no tokens", NAMES[ty], N, V, flush=True)
        _, x = on_gpu(rows_of(ty, N, V))
        X = f64(x)
        _, m, ls, H = ref_logp(X, 0.8)
        lse2 = t.tensor(np.stack([m, ls], 1), dtype=t.float32, device="cuda")
        ent = t.tensor(H, dtype=t.float32, device="cuda")
        g = t.Generator().manual_seed(V)
        a, b = (t.randn(N, generator=g).cuda() for _ in range(2))
        for dlse, dent in ((a, None), (None, b), (a, b)):
            _, d = like_rows(x, ty)
            logprobs_bwd(lib, x, ty, 0.8, None, lse2, ent, None, dlse, dent, d)
            c0, c1 = (np.zeros(N) if v is None else f64(v) for v in (dlse, dent))
            want = ref_bwd(X, 0.8, np.zeros((N, 0), int), np.zeros((N, 0)), c0, c1)
            close(f64(d), want, grad_tol(ty, X, 0.8, want, np.abs(c0), c1, H, 0.8), "dlogits")


def test_logprobs_bwd_masked_tokens(lib):
    """A masked token that is not given has gradient 0 exactly."""
    t = _t()
    for ty in (F32, F16, BF16):
        for N, V in ((4, 300), (4, 70001), (600, 2048)):
            _, x = on_gpu(rows_of(ty, N, V))
            x[:, : V // 2] = -math.inf
            ids = some_ids(N, V, 2, 4, none=False)
            f = logprobs(lib, x, ty, 1.0, ids, 0)
            dlogp, dent = t.randn(N, 2, device="cuda"), t.randn(N, device="cuda")
            _, d = like_rows(x, ty)
            logprobs_bwd(lib, x, ty, 1.0, ids, f.lse2, f.entropy, dlogp, None, dent, d)
            assert bool(d.isfinite().all())
            d.scatter_(1, ids.long(), 0.0)
            assert not bool(d[:, : V // 2].any()) and bool(d[:, V // 2:].any(1).all())


@pytest.mark.parametrize("ty,N,V", [(F32, 70, 2048), (BF16, 9, 5003), (F32, 2, 70000), (F16, 45, 60001)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_without_losses(lib, ty, N, V, tail):
    """rows and loss NULL: the same gradient."""
    t = _t()
    print("no losses", NAMES[ty], N, V, tail, flush=True)
    _, x = on_gpu(rows_of(ty, N, V))
    ids, tl = teacher(x, 20, 2.0)
    tgt = some_ids(N, V, 1, 5)
    _, d = like_rows(x, ty)
    distill(lib, x, ty, ids, tl, tail, 2.0, 1.0, tgt, 0.5, d)
    _, d2 = like_rows(x, ty)
    nb = lib.tlg_distill_ws_bytes(ty, N, V)
    ws = t.full((nb + 16,), 255, device="cuda", dtype=t.uint8)
    lib.distill(x.data_ptr(), ty, V, N, V, ids.data_ptr(), tl.data_ptr(), 20, int(tail), 2.0, 1.0, tgt.data_ptr(), 0.5,
                None, None, d2.data_ptr(), V, 1.0, ws.data_ptr(), nb, stream())
    assert t.equal(d, d2)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,V,tau", [(9, 300, 1.0), (70, 2048, 2.0), (2100, 1000, 2.0), (45, 50003, 1.0)])
def test_distill_weights_of_either_sign(lib, N, V, tau, tail):
    """Zero and negative weights: negating both negates every bit of the results,
    and each term alone counts as it does beside the other."""
    t = _t()
    print("weights", N, V, tau, tail, flush=True)
    _, x = on_gpu(rows_of(F32, N, V))
    ids, tl = teacher(x, 12, tau)
    tgt = t.randint(0, V, (N,), generator=t.Generator().manual_seed(2), dtype=t.int32).cuda()
    tgt[0] = ids[0, 3]

    def run(w_kd, w_ce):
        _, d = like_rows(x, F32)
        o = distill(lib, x, F32, ids, tl, tail, tau, w_kd, tgt, w_ce, d)
        return o, d
    o, d = run(0.75, 0.5)
    n, e = run(-0.75, -0.5)
    assert t.equal(o.rows, -n.rows) and t.equal(o.loss, -n.loss) and t.equal(d, -e)
    X, G, I = f64(x), tgt.cpu().numpy(), ids.cpu().numpy()
    p, p1 = np.exp(ref_logp(X, 1.0 / tau)[0]), np.exp(ref_logp(X, 1.0)[0])
    hot = np.zeros((N, V))
    np.put_along_axis(hot, I.astype(np.int64), 1.0, 1)
    np.put_along_axis(hot, G[:, None].astype(np.int64), 1.0, 1)
    for w_kd, w_ce in ((0.0, 0.5), (-0.75, 0.5), (0.75, -0.5), (0.75, 0.0), (0.0, 0.0)):
        o, d = run(w_kd, w_ce)
        rows, grad = ref_distill(X, I, f64(tl), tail, tau, w_kd, G, w_ce)
        a, b = abs(w_kd), abs(w_ce)
        # |log p| <= 60 here; sums rho-close each, the remainder's three times
        close(f64(o.rows), rows, (a * tau * tau + b) * (3 * rho(V) + 6 * EPS * 120) + 2 * EPS * np.abs(rows), "rows")
        out = 1.0 - np.take_along_axis(p, I.astype(np.int64), 1).sum(1)
        ratio = 2.0 + (1.0 / out if tail else 0.0 * out)
        bar = (a * tau * p * ratio[:, None] + b * p1) * (EPS * (4 * 120 + 12) + 4 * rho(V)) + 8 * EPS * (a * tau + b) * hot
        close(f64(d), grad, bar + 8 * EPS * np.abs(grad) + tiny(F32), "dlogits")


# ------------------------------------------------- graphs, streams, repeats --
@pytest.mark.parametrize("N,V", [(2, 60000), (40, 2048), (600, 3001)])
def test_same_bits_every_time(lib, N, V):
    """Equal calls give equal bits, whatever the workspace held before."""
    t = _t()
    for ty in (F32, BF16):
        _, x = on_gpu(rows_of(ty, N, V))
        ids = some_ids(N, V, 2, 1)
        a, b = logprobs(lib, x, ty, 1.0, ids, 30, 255), logprobs(lib, x, ty, 1.0, ids, 30, 0)
        for n in ("logp", "lse2", "entropy", "top_ids", "top_logp"):
            assert t.equal(getattr(a, n).nan_to_num(7.0), getattr(b, n).nan_to_num(7.0)), n
        tids, tl = teacher(x, 16, 1.0)
        _, d1 = like_rows(x, ty)
        _, d2 = like_rows(x, ty)
        p, q = (distill(lib, x, ty, tids, tl, True, 1.0, 1.0, None, 0.0, d, ws_fill=f)
                for d, f in ((d1, 255), (d2, 0)))
        assert t.equal(d1, d2) and t.equal(p.rows, q.rows) and t.equal(p.loss, q.loss)


@pytest.mark.parametrize("N,V", [(1, 60000), (48, 2048), (600, 3001)])
def test_scoring_then_distillation_captured(lib, N, V):
    """A teacher's scores into a student's distillation and a policy gradient,
    captured once and replayed with new logits between eager calls: every
    replay equals the eager chain bit for bit."""
    t = _t()
    ty, K = BF16, 12
    tx, sx = (t.empty(N, V, dtype=t.bfloat16, device="cuda") for _ in range(2))
    ids = some_ids(N, V, 1, 3)
    f = dict(device="cuda")
    dlogp = t.full((N, 1), -1.0 / N, **f)
    dent = t.full((N,), -0.01 / N, **f)

    class B:
        def __init__(self):
            self.logp, self.lse2, self.ent = t.zeros(N, 1, **f), t.zeros(N, 2, **f), t.zeros(N, **f)
            self.ti, self.tl = t.zeros(N, K, dtype=t.int32, **f), t.zeros(N, K, **f)
            self.rows, self.loss = t.zeros(N, **f), t.zeros(1, **f)
            self.d, self.d2 = t.zeros(N, V, dtype=t.bfloat16, **f), t.zeros(N, V, dtype=t.bfloat16, **f)
            self.nb = lib.tlg_logprobs_ws_bytes(ty, N, V, K)
            self.nk = lib.tlg_distill_ws_bytes(ty, N, V)
            self.ws = t.zeros(max(self.nb, self.nk) + 16, dtype=t.uint8, **f)

        def run(self):
            st = stream()
            lib.logprobs(tx.data_ptr(), ty, V, N, V, 0.5, None, 0, None, None, None, K, self.ti.data_ptr(),
                         self.tl.data_ptr(), self.ws.data_ptr(), self.nb, st)
            lib.distill(sx.data_ptr(), ty, V, N, V, self.ti.data_ptr(), self.tl.data_ptr(), K, 1, 2.0, 1.0, None, 0.0,
                        self.rows.data_ptr(), self.loss.data_ptr(), self.d.data_ptr(), V, 1.0 / N,
                        self.ws.data_ptr(), self.nk, st)
            lib.logprobs(sx.data_ptr(), ty, V, N, V, 1.0, ids.data_ptr(), 1, self.logp.data_ptr(),
                         self.lse2.data_ptr(), self.ent.data_ptr(), 0, None, None, self.ws.data_ptr(), self.nb, st)
            lib.logprobs_bwd(sx.data_ptr(), ty, V, N, V, 1.0, ids.data_ptr(), 1, self.lse2.data_ptr(),
                             self.ent.data_ptr(), dlogp.data_ptr(), None, dent.data_ptr(), self.d2.data_ptr(), V, st)

        def all(self):
            return [self.logp, self.lse2, self.ent, self.ti, self.tl, self.rows, self.loss, self.d, self.d2]
    cap, eager = B(), B()
    tx.normal_()
    sx.normal_()
    cap.run()
    t.cuda.synchronize()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g):
        cap.run()
    for seed in range(4):
        t.manual_seed(seed)
        sx.copy_(2.5 * t.randn(N, V, device="cuda"))
        tx.copy_(sx.float() + 0.5 * t.randn(N, V, device="cuda"))
        for a in cap.all():
            a.zero_()
        g.replay()
        t.cuda.synchronize()
        eager.run()
        t.cuda.synchronize()
        for a, b in zip(cap.all(), eager.all()):
            assert t.equal(a, b)
    # and the chain is right: the student's loss falls along its own gradient
    o = cap
    assert bool((o.rows >= -1e-5).all()) and float(o.loss) > 0


def test_calls_on_two_streams_at_once(lib):
    """Calls with workspaces of their own on two streams at the same time."""
    t = _t()
    N, V, K = 3, 70000, 40
    _, x = on_gpu(rows_of(F32, N, V))
    _, y = on_gpu(rows_of(F32, N, V, seed=9))
    want = [logprobs(lib, z, F32, 1.0, None, K) for z in (x, y)]
    t.cuda.synchronize()
    s = [t.cuda.Stream(), t.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, z in enumerate((x, y)):
            with t.cuda.stream(s[i]):
                got[i].append(logprobs(lib, z, F32, 1.0, None, K))
    t.cuda.synchronize()
    for i in (0, 1):
        for o in got[i]:
            assert t.equal(o.top_ids, want[i].top_ids) and t.equal(o.lse2, want[i].lse2)
            assert t.equal(o.top_logp, want[i].top_logp) and t.equal(o.entropy, want[i].entropy)


def test_rows_behind_four_gigabytes(lib):
    """Row offsets beyond 32 bits of bytes: the last rows of a tall buffer."""
    t = _t()
    N, V, ld = 3, 5000, 1 << 30
    buf = t.empty((N - 1) * ld + V, dtype=t.bfloat16, device="cuda")
    x = t.as_strided(buf, (N, V), (ld, 1))
    x.copy_(2.5 * t.randn(N, V, device="cuda"))
    ids = some_ids(N, V, 1, 1, none=False)
    o = logprobs(lib, x, BF16, 1.0, ids, 7)
    check_logprobs(o, x, 1.0, ids, 7)
    d = t.empty(N, V, dtype=t.bfloat16, device="cuda")
    dlogp = t.randn(N, 1, device="cuda")
    logprobs_bwd(lib, x, BF16, 1.0, ids, o.lse2, o.entropy, dlogp, None, None, d)
    small = x.contiguous()
    d2 = t.empty_like(d)
    logprobs_bwd(lib, small, BF16, 1.0, ids, o.lse2, o.entropy, dlogp, None, None, d2)
    assert t.equal(d, d2)
    logprobs_bwd(lib, x, BF16, 1.0, ids, o.lse2, o.entropy, dlogp, None, None, x)          # and written there
    assert t.equal(x.contiguous(), d)
