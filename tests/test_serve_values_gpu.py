"""GPU tests of what attention over a paged cache (include/tlserve.h) makes of values:
how many bits its weights keep, and what rows get of NaN and infinities that they see.

Tolerances.  eps = 2^-24.  A score is off by (hd + 1) eps sum_d |q_d k_d| scale, its
weight by that, the same of the row's maximum, and eps (4 |s - m| + 6) of the exponent:
d_t.  16-bit rows have weights of two pieces, off by WEIGHT(type) more (twice the type's
half step) and, for fp16, whose smallest step is 2^-24, by SMALL of the row's
largest.  A sum of L terms in any order adds (L + 64) eps, numerator and
denominator each, and what is written its own half step:
  sum_t p_t |v_t| (2 d_t + WEIGHT + 2 (L + 64) eps) + SMALL sum_t |v_t| + half |out|
"""
import math

import numpy as np
import pytest

from test_serve_gpu import _t, BF16, EPS, F16, F32, NAMES, PAIR_IDS, PAIRS, Seqs, check, dtype, half, ints, queries, run_attn, tiny

pytestmark = pytest.mark.gpu
WEIGHT = {F32: 0.0, F16: 2.0 ** -22, BF16: 2.0 ** -16}
SMALL = {F32: 0.0, F16: 2.0 ** -36, BF16: 0.0}


def reference(s, q, H, type, scale, win, sinks):
    """out [N][H][hd] in float64 and its bound.  Values that are not finite count for the
    rows that see them, whatever their weight: NaN, or infinities of one sign."""
    G = H // s.KV
    out, tol = np.full((s.N, H, s.hd), np.nan), np.zeros((s.N, H, s.hd))
    for b, (n, L) in enumerate(zip(s.rows, s.lens)):
        r0 = int(s.row0[b])
        pos, tt = np.arange(L - n, L)[:, None], np.arange(L)[None]
        see = tt <= pos
        if win:
            see &= (tt > pos - win) | (tt < sinks)
        k, v = s.get(s.K, b, L).numpy(), s.get(s.V, b, L).numpy()
        for h in range(H):
            qq, kk, vv = q[r0:r0 + n, h], k[:, h // G], v[:, h // G]
            z = np.where(see, scale * (qq @ kk.T), -np.inf)
            mag = np.where(see, scale * (abs(qq) @ abs(kk).T), 0.0)
            m = z.max(1, keepdims=True)
            e = np.exp(z - m)
            p = e / e.sum(1, keepdims=True)
            d = (s.hd + 1) * EPS * (mag + mag.max(1, keepdims=True)) + EPS * (4 * np.where(see, m - z, 0.0) + 6)
            ok = np.isfinite(vv)
            w = np.where(ok, vv, 0.0)
            o = p @ w
            t = (p * (2 * d + WEIGHT[type] + 2 * (L + 64) * EPS)) @ abs(w) + SMALL[type] * (see @ abs(w)) + \
                half(type) * abs(o) + tiny(type)
            nan, up, down = (see.astype(float) @ x.astype(float) > 0 for x in (np.isnan(vv), vv == np.inf, vv == -np.inf))
            o = np.where(nan | (up & down), np.nan, np.where(up, np.inf, np.where(down, -np.inf, o)))
            out[r0:r0 + n, h], tol[r0:r0 + n, h] = o, t
    return out, tol


def compare(lib, s, H, type, scale, win=0, sinks=0, q=None):
    q = queries(s, H, type) if q is None else q
    out, _ = run_attn(lib, s, q, H, type, scale, win, sinks)
    want, tol = reference(s, q.double().numpy(), H, type, scale, win, sinks)
    inside = np.zeros(s.N, bool)
    inside[int(s.row0[0]):int(s.row0[-1])] = True
    check(out.cpu().double().numpy().reshape(s.N, H, s.hd)[inside], want[inside], tol[inside], "out")


@pytest.mark.parametrize("type", [F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("rows,lens,KV,H,hd,page,win", [
    ([128], [700], 1, 1, 32, 16, 0), ([150, 40], [600, 300], 2, 8, 64, 16, 0), ([70, 64], [400, 130], 1, 4, 96, 7, 0),
    ([100, 90], [900, 90], 2, 8, 128, 64, 0), ([100], [500], 2, 4, 128, 7, 130), ([80], [333], 1, 2, 256, 16, 0),
    ([1, 3], [900, 200], 2, 8, 128, 16, 0)])
def test_weights_keep_twice_their_bits(lib, type, rows, lens, KV, H, hd, page, win):
    """Rounded to the rows' type once, weights are off by 2^-8 (bf16): more than the
    output's own rounding wherever values cancel."""
    s = Seqs(rows, lens, KV, hd, page, type, lead=1, tail=1).gpu()
    compare(lib, s, H, type, hd ** -0.5, win, 3 if win else 0)


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "minus"])
@pytest.mark.parametrize("H,rows,lens,hd,page,win", [
    (1, [256], [256], 64, 16, 0), (4, [256], [266], 64, 16, 0), (4, [256, 5], [276, 100], 32, 7, 0),
    (8, [256], [276], 64, 7, 0), (1, [256], [300], 128, 16, 200), (4, [100], [310], 96, 16, 200),
    (8, [60], [300], 256, 16, 150), (4, [100], [200], 64, 16, 30)])
def test_visible_values_of_many_rows(lib, type, kv, value, H, rows, lens, hd, page, win):
    """One element of some tokens' values is not finite: rows that see the token get it
    whether its tile is seen whole or in part by them, by their wave or by the rows that share
    their workgroup; the others' are as ever."""
    spoiled(lib, type, kv, value, H, rows, lens, hd, page, win)


def spoiled(lib, type, kv, value, H, rows, lens, hd, page, win):
    s = Seqs(rows, lens, 1, hd, page, kv)
    for b, (n, L) in enumerate(zip(rows, lens)):
        for i, pos in enumerate((1, 10, 40, L - n + 3, L - n // 2, L - 70, L - 1)):
            if 0 <= pos < L:
                g, o = s.slots(b, np.array([pos]))
                x = s.V[g, o]
                x[..., 5 + 3 * i] = value if i < 6 else -value
                s.V[g, o] = x
    s.gpu()
    compare(lib, s, H, type, hd ** -0.5, win, 2 if win else 0)


@pytest.mark.parametrize("type", [F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "minus"])
@pytest.mark.parametrize("H,start,hd,page", [(4, 7, 64, 16), (1, 31, 128, 7), (8, 3, 32, 16)])
def test_visible_values_of_one_wave(lib, type, value, H, start, hd, page):
    """A tile's last token, which none but rows that see all of the tile see, while others of their
    workgroup see it in part: the 32 columns of a wave begin at position 63 or 127."""
    t = _t()
    s = Seqs([250], [250 + start], 1, hd, page, type)
    for i, pos in enumerate((63, 127)):
        x = t.full((1, 1, hd), 0.5, dtype=s.V.dtype)
        x[..., 9 + 4 * i] = value
        s.put(s.V, 0, np.array([pos]), x)
    s.gpu()
    compare(lib, s, H, type, hd ** -0.5)


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "minus"])
@pytest.mark.parametrize("H,rows,lens,hd,page,win", [
    (1, [1], [200], 32, 16, 0), (4, [1, 3], [300, 77], 64, 7, 0), (8, [1, 2], [2600, 130], 128, 16, 0),
    (4, [5], [400], 96, 16, 200), (4, [2], [150], 256, 16, 0), (2, [9], [100], 64, 16, 30)])
def test_visible_values_of_few_rows(lib, type, kv, value, H, rows, lens, hd, page, win):
    spoiled(lib, type, kv, value, H, rows, lens, hd, page, win)


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows,lens,H", [([1], [1000], 1), ([2, 3], [900, 2600], 4), ([150], [1000], 2)])
def test_small_weights_of_many_tokens(lib, type, kv, rows, lens, H):
    """One token takes nearly all of every row and has the value 0; the others' weights, e^-15
    each and equal, round alike, and their sum is the output."""
    t = _t()
    s = Seqs(rows, lens, 1, 64, 16, kv)
    for b, L in enumerate(lens):
        k = t.zeros(L, 1, 64, dtype=s.K.dtype)
        v = t.full((L, 1, 64), 1000.0, dtype=s.V.dtype)
        k[3, :, 0] = 15.0
        v[3] = 0.0
        s.put(s.K, b, np.arange(L), k)
        s.put(s.V, b, np.arange(L), v)
    s.gpu()
    q = t.zeros(s.N, H, 64, dtype=dtype(type))
    q[..., 0] = 1.0
    compare(lib, s, H, type, 1.0, q=q)


@pytest.mark.parametrize("type,kv", [(F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("N", [32768, 65536])
def test_decreasing_rows_whose_tiles_pass_32_bits(lib, type, kv, N):
    """row0 must not decrease; where it does, so that 512 of 1024 sequences have all rows, their tiles number
    more than 2^31 or 2^32: nothing is taken part in and nothing is written."""
    s = Seqs([1] * 1024, [1] * 1024, 1, 32, 64, kv, extra_ldt=1031)
    s.N = N
    s.gpu()
    s.dev[0].copy_(ints([0, N] * 512 + [0]))
    s.dev[1].fill_(66000)
    s.batch.N, s.batch.max_rows, s.batch.max_len = N, 1, 0
    out, ls = run_attn(lib, s, queries(s, 1, type), 1, type, 0.2)
    assert (out == 7.0).all() and (ls == 7.0).all()


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
def test_decreasing_rows(lib, type, kv):
    """Sequences that share rows, over shares of the batch: any of them may have a row, rows of none
    are left alone."""
    s = Seqs([6, 2, 4], [2600, 2500, 2400], 1, 32, 16, kv, tail=3).gpu()
    s.dev[0].copy_(ints([0, 9, 2, 12]))
    s.batch.max_rows = 2
    out, ls = run_attn(lib, s, queries(s, 2, type), 2, type, 0.2)
    assert (out[12:] == 7.0).all() and (ls[12:] == 7.0).all()


@pytest.mark.parametrize("type,kv", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("rows,lens", [([12, 1, 16], [700, 600, 900]), ([16, 9], [2600, 150]), ([100, 12, 16, 17, 1], [600, 2500, 700, 90, 650])])
def test_rows_around_the_launches_borders(lib, type, kv, hd, rows, lens):
    """32 and 64 columns a sequence and some more and fewer, alone and beside longer chunks, each cut alike
    and shared evenly."""
    s = Seqs(rows, lens, 1, hd, 16, kv, head_major=True, lead=1, tail=1).gpu()
    compare(lib, s, 4, type, hd ** -0.5)
    compare(lib, s, 4, type, hd ** -0.5, 300, 5)
