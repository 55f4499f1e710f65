"""The vocabulary operators: what they compute, on which sizes, and how long.

Three operators over rows of logits [N][V] (include/tltrain.h), as the head
of a model leaves them:

  logprobs      log probabilities of given tokens, the entropy and the K
                likeliest alternatives of every row (tlg_dev_logprobs)
  logprobs_bwd  their gradient with respect to the logits
                (tlg_dev_logprobs_bwd)
  distill       distillation from a teacher's top log probabilities, with the
                hard-target cross-entropy: loss and gradient in one call
                (tlg_dev_distill)

`own` False computes them with elementary tensor operations, True through the
library.  Rows may be wider apart than V (`pad` unused columns) and hold
tokens masked to -inf; a negative token id means "none".
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
BOOSTED = 8                    # likely tokens of a row


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one decoded token's probability and alternatives, the m8 model's head
        dict(name="lp_token", op="logprobs", N=1, V=2048, type="f32", M=1, K=8, temp=1.0, pad=0, masked=False),
        # the same for a large vocabulary, as a server that samples one sequence asks for it
        dict(name="lp_token_wide", op="logprobs", N=1, V=131072, type="bf16", M=1, K=20, temp=1.0, pad=0,
             masked=False),
        # a decode batch under a grammar: most of an odd vocabulary is masked, temperature 0.7
        dict(name="lp_batch", op="logprobs", N=48, V=32003, type="f16", M=1, K=5, temp=0.7, pad=0, masked=True),
        # a teacher's pass over the m3 model's training batch
        dict(name="lp_score", op="logprobs", N=4096, V=2048, type="f32", M=1, K=8, temp=1.0, pad=0, masked=False),
        # scoring long sequences of a large vocabulary with many alternatives: the largest forward
        dict(name="lp_large", op="logprobs", N=4096, V=131072, type="bf16", M=1, K=32, temp=1.0, pad=0,
             masked=False),
        # policy gradient with an entropy bonus on the m3 model's batch
        dict(name="lpb_batch", op="logprobs_bwd", N=4096, V=2048, type="f32", M=1, temp=1.0, pad=0, masked=False),
        # several candidate tokens a row, odd vocabulary in padded rows, padded batch
        dict(name="lpb_odd", op="logprobs_bwd", N=509, V=50021, type="f16", M=4, temp=1.3, pad=11, masked=True),
        # the largest gradient
        dict(name="lpb_large", op="logprobs_bwd", N=4096, V=131072, type="bf16", M=1, temp=1.0, pad=0, masked=False),
        # distilling a short sequence into the nano model
        dict(name="kd_small", op="distill", N=64, V=2048, type="f32", K=8, tail=False, temp=1.0, w_kd=1.0, w_ce=0.0,
             pad=0, masked=False),
        # the m3 model's batch: soft targets at temperature 2 with the hard ones
        dict(name="kd_batch", op="distill", N=4096, V=2048, type="f32", K=32, tail=False, temp=2.0, w_kd=0.7,
             w_ce=0.3, pad=0, masked=False),
        # an odd vocabulary in padded rows, the teacher's remaining mass as one more outcome
        dict(name="kd_odd", op="distill", N=301, V=50021, type="f32", K=50, tail=True, temp=1.0, w_kd=1.0, w_ce=0.5,
             pad=11, masked=True),
        # the largest: a long batch of a large vocabulary
        dict(name="kd_large", op="distill", N=4096, V=131072, type="bf16", K=64, tail=True, temp=1.0, w_kd=1.0,
             w_ce=0.0, pad=0, masked=False),
    ]


def _gscale(case):
    """What a mean over the rows multiplies the gradients with; fp16 gradients
    are scaled up, as a program that keeps them in fp16 does."""
    return (4096.0 if case["type"] == "f16" else 1.0) / case["N"]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs_bwd", "distill"])
    V = rng.choice([2048, _log(rng, 1024, 131072), _log(rng, 1024, 131072) // 8 * 8])
    most = min(8192, (1 << 28) // V)
    c = dict(op=op, N=_log(rng, 1, most), V=V, type=rng.choice(["f32", "f16", "bf16"]),
             temp=rng.choice([1.0, 1.0, 0.7, 2.0]), pad=rng.choice([0, 0, 0, 8, rng.randint(1, 64)]),
             masked=rng.random() < 0.25)
    if op == "distill":
        c.update(K=_log(rng, 1, 128), tail=rng.random() < 0.4, w_kd=rng.choice([1.0, 0.5]),
                 w_ce=rng.choice([0.0, 0.5]))
    else:
        c.update(M=rng.choice([1, 1, 1, 2, 5]))
        if op == "logprobs":
            c.update(K=rng.choice([0, 1, 5, 20, _log(rng, 1, 64)]))
    return c


# ---------------------------------------------------------------- prepare --
def _inputs(case, seed):
    """The seeded inputs of a case: logits of a head (a spread of about 2 with
    a few likely tokens a row), token ids, and for distill a teacher that
    mostly agrees with the student."""
    c = case
    N, V, dt = c["N"], c["V"], TYPES[c["type"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = V + c["pad"]
    x = torch.randn(N, ld, generator=g, device="cuda").mul_(2.0)
    likely = torch.randint(0, V, (N, BOOSTED), generator=g, device="cuda")
    x.scatter_add_(1, likely, 3.0 + 5.0 * torch.rand(N, BOOSTED, generator=g, device="cuda"))
    s = {}
    if c["op"] == "distill":
        K = c["K"]
        teacher = x[:, :V] + 0.5 * torch.randn(N, V, generator=g, device="cuda")
        teacher = teacher / c["temp"]
        lse = torch.logsumexp(teacher, 1, keepdim=True)
        v, i = torch.topk(teacher, K, dim=1)
        s.update(t_ids=i.int().contiguous(), t_logp=(v - lse).contiguous())
        del teacher
        s["tgt"] = likely[:, 0].int().contiguous()
        if c["masked"]:                  # a padded batch: its last rows have neither teacher nor target
            s["t_ids"][N - N // 8:] = -1
            s["tgt"][N - N // 8:] = -1
    else:
        M = c["M"]
        ids = torch.randint(0, V, (N, M), generator=g, device="cuda")
        ids[:, 0] = likely[:, 0]
        if c["masked"]:
            # a grammar leaves about one token in four, the asked ones among them
            drop = torch.rand(N, V, generator=g, device="cuda") < 0.75
            drop.scatter_(1, ids, False)
            x[:, :V].masked_fill_(drop, -math.inf)
            ids[N - N // 8:] = -1
        s["ids"] = ids.int().contiguous()
        if c["op"] == "logprobs_bwd":
            s["dlogp"] = torch.randn(N, M, generator=g, device="cuda") * _gscale(c)
            s["dlse"] = 1e-3 * torch.randn(N, generator=g, device="cuda") * _gscale(c)
            s["dent"] = torch.full((N,), -0.01 * _gscale(c), device="cuda")
    buf = x.to(dt)
    if c["pad"]:
        buf[:, V:] = 100.0               # columns behind the vocabulary hold something else
    s["logits"] = buf[:, :V]
    return s


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    c, N, V = case, case["N"], case["V"]
    if c["op"] == "logprobs_bwd":        # what the forward pass left
        st = _stats(s["logits"], 1.0 / c["temp"])
        s.update(lse2=torch.stack([st[0], st[1]], 1).contiguous(), entropy=st[2])
    if own:
        s["lib"] = _lib()
        lib, code = s["lib"], CODES[c["type"]]
        f = dict(device="cuda", dtype=torch.float32)
        if c["op"] == "logprobs":
            s.update(logp=torch.empty(N, c["M"], **f), lse2=torch.empty(N, 2, **f), entropy=torch.empty(N, **f),
                     top_ids=torch.empty(N, c["K"], device="cuda", dtype=torch.int32),
                     top_logp=torch.empty(N, c["K"], **f))
            nb = lib.tlg_logprobs_ws_bytes(code, N, V, c["K"])
        else:
            s["dlogits"] = torch.empty(N, s["logits"].stride(0), device="cuda", dtype=TYPES[c["type"]])[:, :V]
            nb = 0
            if c["op"] == "distill":
                s.update(rows=torch.empty(N, **f), loss=torch.empty(1, **f))
                nb = lib.tlg_distill_ws_bytes(code, N, V)
        s["ws"] = torch.empty(max(nb, 16), device="cuda", dtype=torch.uint8)
        s["ws_bytes"] = nb
    return s


def _lib():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinylm-c_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tlgemm
    lib = tlgemm.load()
    lib.check(lib.tlg_init(torch.cuda.current_device()), "tlg_init")
    return lib


# -------------------------------------------------------------------- run --
def run(state):
    op = state["case"]["op"]
    return (_own if own else _plain)[op](state)


def _own_logprobs(s):
    c, x, st = s["case"], s["logits"], torch.cuda.current_stream().cuda_stream
    s["lib"].logprobs(x.data_ptr(), CODES[c["type"]], x.stride(0), c["N"], c["V"], 1.0 / c["temp"],
                      s["ids"].data_ptr(), c["M"], s["logp"].data_ptr(), s["lse2"].data_ptr(),
                      s["entropy"].data_ptr(), c["K"], s["top_ids"].data_ptr(), s["top_logp"].data_ptr(),
                      s["ws"].data_ptr(), s["ws_bytes"], st)
    return [s["logp"], s["lse2"], s["entropy"], s["top_ids"], s["top_logp"]]


def _own_logprobs_bwd(s):
    c, x, d, st = s["case"], s["logits"], s["dlogits"], torch.cuda.current_stream().cuda_stream
    s["lib"].logprobs_bwd(x.data_ptr(), CODES[c["type"]], x.stride(0), c["N"], c["V"], 1.0 / c["temp"],
                          s["ids"].data_ptr(), c["M"], s["lse2"].data_ptr(), s["entropy"].data_ptr(),
                          s["dlogp"].data_ptr(), s["dlse"].data_ptr(), s["dent"].data_ptr(), d.data_ptr(),
                          d.stride(0), st)
    return [d]


def _own_distill(s):
    c, x, d, st = s["case"], s["logits"], s["dlogits"], torch.cuda.current_stream().cuda_stream
    s["lib"].distill(x.data_ptr(), CODES[c["type"]], x.stride(0), c["N"], c["V"], s["t_ids"].data_ptr(),
                     s["t_logp"].data_ptr(), c["K"], int(c["tail"]), c["temp"], c["w_kd"], s["tgt"].data_ptr(),
                     c["w_ce"], s["rows"].data_ptr(), s["loss"].data_ptr(), d.data_ptr(), d.stride(0),
                     _gscale(c), s["ws"].data_ptr(), s["ws_bytes"], st)
    return [s["rows"], s["loss"], d]


def _stats(logits, scale):
    """max, log sum exp(scale (x - max)) and entropy of every row, fp32."""
    x = logits.float()
    m = x.max(1, keepdim=True).values
    z = (x - m).mul_(scale)
    e = z.exp()
    s = e.sum(1, keepdim=True)
    u = torch.where(e > 0, z * e, 0.0).sum(1, keepdim=True)
    return m[:, 0], s.log()[:, 0], (s.log() - u / s)[:, 0]


def _plain_logprobs(s):
    c, scale, K = s["case"], 1.0 / s["case"]["temp"], s["case"]["K"]
    x = s["logits"].float()
    m, ls, ent = _stats(x, scale)
    ids = s["ids"].long()
    picked = x.gather(1, ids.clamp_min(0))
    logp = torch.where(ids < 0, 0.0, (picked - m[:, None]) * scale - ls[:, None])
    top_ids = torch.empty(c["N"], K, device="cuda", dtype=torch.int32)
    top_logp = torch.empty(c["N"], K, device="cuda")
    rest = x.clone() if K else x
    for k in range(K):                   # the largest of what is left, the first one of equals
        i = rest.argmax(1, keepdim=True)
        v = rest.gather(1, i)
        rest.scatter_(1, i, -math.inf)
        top_ids[:, k] = torch.where(v > -math.inf, i, -1)[:, 0].int()
        top_logp[:, k] = ((v - m[:, None]) * scale - ls[:, None])[:, 0]
    return [logp, torch.stack([m, ls], 1), ent, top_ids, top_logp]


def _plain_logprobs_bwd(s):
    c, scale = s["case"], 1.0 / s["case"]["temp"]
    x = s["logits"].float()
    logp = (x - s["lse2"][:, :1]) * scale - s["lse2"][:, 1:]
    p = logp.exp()
    ids = s["ids"].long()
    g = torch.where(ids < 0, 0.0, s["dlogp"])
    d = p * (s["dlse"] - g.sum(1))[:, None]
    d -= torch.where(p > 0, p * (logp + s["entropy"][:, None]), 0.0) * s["dent"][:, None]
    d.scatter_add_(1, ids.clamp_min(0), g)
    return [(d * scale).to(TYPES[c["type"]])]


def _plain_distill(s):
    c, tau, N = s["case"], s["case"]["temp"], s["case"]["N"]
    x = s["logits"].float()
    m = x.max(1, keepdim=True).values
    p = (x - m).div_(tau).exp_()
    total = p.sum(1, keepdim=True)
    p /= total
    ids, have = s["t_ids"].long(), s["t_ids"] >= 0
    at = ids.clamp_min(0)
    # the teacher's side in 64 bits: what its K entries leave over, and a small
    # divergence as a difference of large terms
    q = torch.where(have, s["t_logp"].double().exp(), 0.0)
    logp = (x.gather(1, at) - m).double() / tau - total.double().log()
    rows = torch.zeros(N, device="cuda", dtype=torch.float64)
    if c["tail"]:
        inside = torch.zeros_like(x).scatter_add_(1, at, have.float()) > 0
        pr = torch.where(inside, 0.0, p).sum(1).double()
        qr = torch.where(have.any(1), (1.0 - q.sum(1)).clamp_min(0.0), 0.0)
        rows += torch.where(qr > 0, qr * (qr.log() - pr.log()), 0.0)
        mass = q.sum(1) + qr
        ratio = torch.where(qr > 0, qr / pr, 0.0)
        d = p * torch.where(inside, mass.float()[:, None], (mass - ratio).float()[:, None])
    else:
        q = q / q.sum(1, keepdim=True).clamp_min(1e-30)
        d = p * q.sum(1, keepdim=True).float()
    rows += torch.where(q > 0, q * (q.log() - logp), 0.0).sum(1)
    rows *= c["w_kd"] * tau * tau
    d.scatter_add_(1, at, -q.float())
    d *= c["w_kd"] * tau
    if c["w_ce"]:
        e1 = (x - m).exp_()
        total1 = e1.sum(1, keepdim=True)
        t = s["tgt"].long()[:, None]
        on = t >= 0
        z = (x.gather(1, t.clamp_min(0)) - m).double() - total1.double().log()
        rows += torch.where(on, -z, 0.0)[:, 0] * c["w_ce"]
        d += torch.where(on, e1 / total1, 0.0) * c["w_ce"]
        d.scatter_add_(1, t.clamp_min(0), -c["w_ce"] * on.float())
    return [rows.float(), rows.mean().float().reshape(1), (d * _gscale(c)).to(TYPES[c["type"]])]


_own = dict(logprobs=_own_logprobs, logprobs_bwd=_own_logprobs_bwd, distill=_own_distill)
_plain = dict(logprobs=_plain_logprobs, logprobs_bwd=_plain_logprobs_bwd, distill=_plain_distill)


# ------------------------------------------------------------------- work --
def work(case):
    """Logits read once, everything the call returns written once; an
    exponential, a product or two and the sums for every logit."""
    c = case
    N, V, b = c["N"], c["V"], 4 if c["type"] == "f32" else 2
    if c["op"] == "logprobs":
        return dict(bytes=N * V * b + N * (8 * c["M"] + 12 + 8 * c["K"]), flops=6 * N * V)
    if c["op"] == "logprobs_bwd":
        return dict(bytes=2 * N * V * b + N * (8 * c["M"] + 20), flops=8 * N * V)
    return dict(bytes=2 * N * V * b + N * (8 * c["K"] + 12) + 4, flops=10 * N * V)


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    """What run returns, from the definitions in 64 bits, some rows at a time."""
    s = _inputs(case, seed)
    N, V = case["N"], case["V"]
    step = max(1, (1 << 26) // V)
    parts = []
    for r in range(0, N, step):
        part = {k: (v[r:r + step] if torch.is_tensor(v) else v) for k, v in s.items()}
        parts.append(_exact[case["op"]](case, part))
    out = [torch.cat(col) for col in zip(*parts)]
    if case["op"] == "distill":
        out.insert(1, out[0].mean().reshape(1))
    return out


def _log_softmax64(z):
    top = z.amax(1, keepdim=True)
    return z - (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))


def _entropy64(lp):
    p = torch.exp(lp)
    return -(p * lp.masked_fill(p == 0, 0.0)).sum(1)


def _one_hot_sum(ids, weight, V):
    """sum_j weight[n][j] [v = ids[n][j]], negative ids left out, [N][V]."""
    out = torch.zeros(ids.shape[0], V + 1, device=ids.device, dtype=torch.float64)
    out.scatter_add_(1, torch.where(ids < 0, V, ids), weight.double())
    return out[:, :V]


def _exact_logprobs(c, s):
    x = s["logits"].double()
    lp = _log_softmax64(x / c["temp"])
    ids = s["ids"].long()
    logp = torch.gather(lp, 1, ids.clamp_min(0)).masked_fill(ids < 0, 0.0)
    top = x.amax(1)
    ls = torch.log(torch.exp((x - top[:, None]) / c["temp"]).sum(1))
    # order by value, the lower index first among equals: one whole number for both
    bits = s["logits"].float().contiguous().view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=x.device))
    top_ids = torch.topk(key, c["K"], dim=1, sorted=True).indices if c["K"] else ids[:, :0]
    top_logp = torch.gather(lp, 1, top_ids)
    return [logp, torch.stack([top, ls], 1), _entropy64(lp),
            top_ids.masked_fill(top_logp == -math.inf, -1).int(), top_logp]


def _exact_logprobs_bwd(c, s):
    scale = 1.0 / c["temp"]
    lp = _log_softmax64(s["logits"].double() * scale)
    p, ids = torch.exp(lp), s["ids"].long()
    want = _one_hot_sum(ids, s["dlogp"], c["V"])
    d = want - p * want.sum(1, keepdim=True) + p * s["dlse"].double()[:, None]
    inner = lp.masked_fill(p == 0, 0.0) + _entropy64(lp)[:, None]
    return [scale * (d - s["dent"].double()[:, None] * p * inner)]


def _exact_distill(c, s):
    tau, V, x = c["temp"], c["V"], s["logits"].double()
    lp = _log_softmax64(x / tau)
    p, ids = torch.exp(lp), s["t_ids"].long()
    real = ids >= 0
    q = torch.exp(s["t_logp"].double()) * real
    some = real.any(1).double()
    if not c["tail"]:
        q = q / q.sum(1, keepdim=True).clamp_min(1e-300)
    full = _one_hot_sum(ids, q, V)
    rows = torch.where(full > 0, full * (torch.log(full.clamp_min(1e-300)) - lp), 0.0).sum(1)
    d = p * full.sum(1, keepdim=True) - full
    if c["tail"]:
        support = _one_hot_sum(ids, real.double(), V) > 0
        rest_q = (1.0 - q.sum(1)).clamp_min(0.0) * some
        rest_p = p.masked_fill(support, 0.0).sum(1)
        on = rest_q > 0
        rows += torch.where(on, rest_q * torch.log(rest_q / rest_p), 0.0)
        part = torch.where(on, rest_q / rest_p, 0.0)[:, None]
        d += p * rest_q[:, None] - (p * part).masked_fill(support, 0.0)
    rows, d = rows * c["w_kd"] * tau * tau, d * c["w_kd"] * tau
    if c["w_ce"]:
        t = s["tgt"].long()
        lp1 = _log_softmax64(x)
        on = (t >= 0).double()
        rows += c["w_ce"] * on * -torch.gather(lp1, 1, t.clamp_min(0)[:, None])[:, 0]
        d += c["w_ce"] * (torch.exp(lp1) * on[:, None] - _one_hot_sum(t[:, None], on[:, None], V))
    return [rows, d * _gscale(c)]


_exact = dict(logprobs=_exact_logprobs, logprobs_bwd=_exact_logprobs_bwd, distill=_exact_distill)
