"""Sampled self-speculative generation (tl_decode_sample_spec) on a ring that has fewer
slots than the text has positions, against a decoder fed one token at a time."""
import numpy as np
import pytest

import tlgemm
from test_serve_chain_gpu import KW, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def host(lib):
    return tlgemm.host()


@pytest.fixture(scope="module")
def stream(lib):
    return lib.tlg_stream_create()


@pytest.mark.parametrize("f16", [0, 1])
@pytest.mark.parametrize("n_mtp,mmax,extra", [
    (3, 8, {}), (1, 2, {}), (0, 4, {}), (3, 8, dict(win=20)), (3, 8, dict(win=30)), (3, 8, dict(win=20, full_every=2)),
    (7, 8, dict(win=28))])
def test_sample_spec_on_a_wrapped_ring(lib, host, stream, n_mtp, mmax, extra, f16):
    """Every token's log probability is that of the row before it with nothing drafted:
    drafted rows take no slot of a token that a row still sees."""
    kw, W, maxpos = dict(KW, n_mtp=n_mtp, **extra), 32, 96
    m, P = weights(kw, 11)
    # heads that draft what the model is likely to say next, so that some are kept
    prompt, temp = np.arange(3, 14, dtype=np.int32), 0.7
    n = maxpos - len(prompt) + 1
    a = host.decode(kw, W, kv_f16=f16, exact_exp=1, maxpos=maxpos, mmax=mmax)
    b = host.decode(kw, W, kv_f16=f16, exact_exp=1, maxpos=maxpos, mmax=1)
    a.upload(P, stream)
    b.upload(P, stream)
    toks, lp, chunks = a.sample_spec(prompt, n, stream, temp=temp, seed=5)
    assert n - 1 >= chunks >= (n - 1) / (min(n_mtp, mmax - 1) + 1)
    for i, tok in enumerate(prompt):
        z = b.chunk(np.array([tok], np.int32), i, stream)[0]
    for i, tok in enumerate(toks):
        x = z.astype(np.float64) / temp
        want = x[tok] - x.max() - np.log(np.exp(x - x.max()).sum())
        # the logits differ by the order of sums alone, and by what that flips of an fp16 ring's roundings
        tol = (2e-5 if not f16 else 2e-3) * abs(x).max() * 2
        assert abs(lp[i] - want) <= tol, (i, lp[i], want)
        if i + 1 < n:
            z = b.chunk(np.array([tok], np.int32), len(prompt) + i, stream)[0]
