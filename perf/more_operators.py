"""The serving operators: what they compute, on which sizes, and how long.

Three operators of a server that decodes a batch of sequences over a paged
KV cache and verifies drafted tokens (include/tlserve.h):

  store   the new rows' keys and values into the cache's pages, RoPE of the
          keys and the queries on the way (tlg_dev_paged_store)
  attn    causal attention of every sequence's new rows over its pages, with a
          sliding window and sink tokens (tlg_dev_paged_attn)
  verify  drafted tokens against the target model's probabilities, and the
          token after the last one kept (tlg_dev_spec_verify)

`own` False computes them with elementary tensor operations, True through the
library.  Sequences are ragged: some have fewer new rows, some none, and their
lengths differ.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BOOSTED = 8                    # likely tokens of a row
ROPE_BASE = 10000.0


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one decoded token of the m8 model into its f16 cache
        dict(name="st_token", op="store", B=1, rows=1, len=200, H=12, KV=3, hd=32, page=16, type="f32", kv="f16",
             fused=False),
        # a batch of drafted chunks whose q, k and v lie in one row of a fused projection
        dict(name="st_batch", op="store", B=61, rows=6, len=2048, H=32, KV=8, hd=128, page=16, type="bf16", kv="bf16",
             fused=True),
        # prompts: the largest
        dict(name="st_prompt", op="store", B=8, rows=2048, len=2048, H=32, KV=8, hd=128, page=64, type="bf16",
             kv="bf16", fused=True),
        # one decoded token of the m8 model at the end of its context: latency
        dict(name="pa_token", op="attn", B=1, rows=1, len=250, H=12, KV=3, hd=32, page=16, type="f32", kv="f16",
             win=0, sinks=0),
        # the m3 model's prompts in its own precision
        dict(name="pa_prompt", op="attn", B=16, rows=256, len=256, H=8, KV=2, hd=32, page=32, type="f32", kv="f32",
             win=0, sinks=0),
        # a decode batch of ragged lengths
        dict(name="pa_batch", op="attn", B=64, rows=1, len=4096, H=32, KV=8, hd=128, page=16, type="bf16", kv="bf16",
             win=0, sinks=0),
        # one long context, one token
        dict(name="pa_long", op="attn", B=1, rows=1, len=131072, H=32, KV=8, hd=128, page=64, type="bf16", kv="bf16",
             win=0, sinks=0),
        # drafted chunks under a sliding window with sinks, pages of an odd size
        dict(name="pa_verify", op="attn", B=32, rows=5, len=8000, H=16, KV=4, hd=64, page=49, type="f16", kv="f16",
             win=1024, sinks=4),
        # the last chunk of a long prompt: the largest
        dict(name="pa_chunk", op="attn", B=1, rows=4096, len=16384, H=32, KV=8, hd=128, page=64, type="bf16",
             kv="bf16", win=0, sinks=0),
        # one sequence's two MTP drafts, the m8 model's head
        dict(name="sv_one", op="verify", B=1, rows=3, V=2048, type="f32", temp=1.0, dtemp=0.0, pad=0, masked=False),
        # a batch under a grammar, odd vocabulary in padded rows, a draft model at another temperature
        dict(name="sv_batch", op="verify", B=48, rows=5, V=32003, type="f16", temp=0.7, dtemp=1.0, pad=11,
             masked=True),
        # the largest: a large vocabulary
        dict(name="sv_large", op="verify", B=256, rows=5, V=131072, type="bf16", temp=1.0, dtemp=1.0, pad=0,
             masked=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attn", "attn", "verify"])
    if op == "verify":
        V = rng.choice([2048, _log(rng, 1024, 131072), _log(rng, 1024, 131072) // 8 * 8])
        rows = rng.randint(1, 9)
        return dict(op=op, B=min(_log(rng, 1, 256), max(1, (1 << 27) // (V * rows))), rows=rows, V=V,
                    type=rng.choice(["f32", "f16", "bf16"]), temp=rng.choice([1.0, 1.0, 0.7, 1.5]),
                    dtemp=rng.choice([0.0, 1.0, 1.0, 0.8]), pad=rng.choice([0, 0, 0, 8, rng.randint(1, 64)]),
                    masked=rng.random() < 0.25)
    KV = rng.choice([1, 2, 3, 4, 8])
    type, kv = rng.choice([("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16")])
    c = dict(op=op, H=KV * rng.choice([1, 2, 4, 4, 5, 8]), KV=KV, hd=rng.choice([32, 64, 64, 96, 128, 128, 256]),
             page=rng.choice([16, 16, 32, 64, 128, rng.randint(5, 100)]), type=type, kv=kv)
    if op == "store":
        c.update(B=_log(rng, 1, 64), rows=_log(rng, 1, 2048), fused=rng.random() < 0.5)
        c["rows"] = max(1, min(c["rows"], (1 << 25) // (c["B"] * (c["H"] + 2 * KV) * c["hd"])))
        c["len"] = c["rows"] + _log(rng, 1, 4096)
        return c
    kind = rng.choice(["token", "draft", "chunk"])
    if kind == "token":
        c.update(B=_log(rng, 1, 128), rows=1, len=_log(rng, 1, 65536))
    elif kind == "draft":
        c.update(B=_log(rng, 1, 64), rows=rng.randint(2, 9), len=_log(rng, 10, 32768))
    else:
        c.update(B=_log(rng, 1, 16), rows=_log(rng, 16, 2048))
        c["len"] = c["rows"] + rng.choice([0, _log(rng, 1, 8192)])
    # no more cached elements nor products than the largest listed cases have
    c["B"] = max(1, min(c["B"], (1 << 28) // (c["len"] * KV * c["hd"])))
    c["B"] = max(1, min(c["B"], (1 << 37) // (c["rows"] * c["len"] * c["H"] * c["hd"])))
    w = rng.choice([0, 0, _log(rng, 16, 4096)])
    c.update(win=w, sinks=rng.choice([0, 4, rng.randint(1, 64)]) if w else 0)
    return c


def _shape(case):
    """New rows and length of every sequence: the first has the most of both,
    of eight later ones one has no new row (a slot whose request ended)."""
    rows, lens = [], []
    for b in range(case["B"]):
        n = case["rows"]
        n = 0 if b % 8 == 5 else n - b * 5 % (n // 2 + 1)
        rows.append(n)
        if case["op"] != "verify":
            lens.append(max(n, case["len"] - b * 40503 % (case["len"] * 3 // 4 + 1)))
    return rows, lens


# ---------------------------------------------------------------- prepare --
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (_verify_inputs if case["op"] == "verify" else _cache_inputs)(case, g)


def _cache_inputs(c, g):
    """A cache whose pages are dealt out in random order, the batch, and the
    rows of its new tokens.  Values are those of the models: N(0, 1)."""
    rows, lens = _shape(c)
    B, KV, hd, page = c["B"], c["KV"], c["hd"], c["page"]
    need = [-(-n // page) for n in lens]
    n_pages, ldt = sum(need) + 1, max(need)
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((B, ldt), -1, device="cuda", dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    row0 = [0]
    for n in rows:
        row0.append(row0[-1] + n)
    N, H = row0[-1], c["H"]
    s = dict(rows=rows, lens=lens, N=N, n_pages=n_pages, ldt=ldt, table=table,
             row0=torch.tensor(row0, dtype=torch.int32).cuda(), len=torch.tensor(lens, dtype=torch.int32).cuda(),
             K=torch.randn(n_pages, page, KV, hd, generator=g, device="cuda").to(TYPES[c["kv"]]),
             V=torch.randn(n_pages, page, KV, hd, generator=g, device="cuda").to(TYPES[c["kv"]]))
    if c["op"] == "attn":
        # queries with a few keys they look for: scores with a spread as heads have it
        s["q"] = (1.5 * torch.randn(N, H, hd, generator=g, device="cuda")).to(TYPES[c["type"]])
        return s
    x = torch.randn(N, (H + 2 * KV) * hd, generator=g, device="cuda").to(TYPES[c["type"]])
    parts = [x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:]]
    s["q"], s["k"], s["v"] = parts if c["fused"] else [p.contiguous() for p in parts]
    s["maxpos"] = max(lens)
    angle = torch.arange(s["maxpos"], device="cuda", dtype=torch.float64)[:, None] * \
        ROPE_BASE ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


def _verify_inputs(c, g):
    """Logits of a target model (a spread of about 2 with a few likely tokens a
    row) and of a draft model that mostly agrees, drafts from the latter,
    uniforms for the tests and exponentials for the token after the last kept."""
    rows, _ = _shape(c)
    B, V, ld = c["B"], c["V"], c["V"] + c["pad"]
    row0 = [0]
    for n in rows:
        row0.append(row0[-1] + n)
    N = row0[-1]
    x = torch.randn(N, ld, generator=g, device="cuda").mul_(2.0)
    x.scatter_add_(1, torch.randint(0, V, (N, BOOSTED), generator=g, device="cuda"),
                   3.0 + 5.0 * torch.rand(N, BOOSTED, generator=g, device="cuda"))
    if c["masked"]:                      # a grammar leaves about one token in four
        drop = torch.rand(N, V, generator=g, device="cuda") < 0.75
        x[:, :V].masked_fill_(drop, -math.inf)
    dt = TYPES[c["type"]]
    y = x + 0.5 * torch.randn(N, ld, generator=g, device="cuda")
    if c["pad"]:
        x[:, V:] = 100.0                 # columns behind the vocabulary hold something else
        y[:, V:] = 100.0
    s = dict(N=N, rows=rows, row0=torch.tensor(row0, dtype=torch.int32).cuda(), x=x.to(dt)[:, :V])
    if c["dtemp"]:
        s["y"] = y.to(dt)[:, :V]
        z = s["y"].float() / c["dtemp"]
        z -= torch.empty_like(z).exponential_(generator=g).log_()
    else:
        z = y[:, :V]
    s["draft"] = z.argmax(1).int()
    for b in range(B):                   # a sequence's last row has nothing to verify
        if rows[b]:
            s["draft"][row0[b + 1] - 1] = -1
    s["u"] = torch.rand(N, generator=g, device="cuda")
    s["noise"] = torch.empty(B, V, device="cuda").exponential_(generator=g).clamp_min_(1e-12)
    return s


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    c, N = case, s["N"]
    if c["op"] == "store":
        s["q_out"] = torch.empty(N, c["H"] * c["hd"], device="cuda", dtype=TYPES[c["type"]])
    if not own:
        return s
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinylm-c_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tlgemm
    s["lib"] = lib = tlgemm.load()
    lib.check(lib.tlg_init(torch.cuda.current_device()), "tlg_init")
    nb = 0
    if c["op"] == "verify":
        s.update(tokens=torch.empty(N, device="cuda", dtype=torch.int32), logp=torch.empty(N, device="cuda"),
                 accepted=torch.empty(c["B"], device="cuda", dtype=torch.int32))
        nb = lib.tlg_spec_verify_ws_bytes(CODES[c["type"]], N, c["V"], c["B"], int(c["dtemp"] > 0))
    else:
        s["pages"] = tlgemm.pages(s["K"].data_ptr(), s["V"].data_ptr(), CODES[c["kv"]], c["KV"], c["hd"], c["page"],
                                  s["n_pages"])
        s["batch"] = tlgemm.batch(c["B"], N, s["row0"].data_ptr(), s["len"].data_ptr(), s["table"].data_ptr(),
                                  s["ldt"], max_rows=c["rows"], max_len=c["len"])
        if c["op"] == "attn":
            s.update(out=torch.empty(N, c["H"], c["hd"], device="cuda", dtype=TYPES[c["type"]]),
                     lse=torch.empty(N, c["H"], device="cuda"))
            nb = lib.paged_attn_ws_bytes(s["pages"], s["batch"], CODES[c["type"]], c["H"])
    s["ws"] = torch.empty(max(nb, 16), device="cuda", dtype=torch.uint8)
    s["ws_bytes"] = nb
    return s


# -------------------------------------------------------------------- run --
def run(state):
    op = state["case"]["op"]
    return (_own if own else _plain)[op](state)


def _own_store(s):
    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    s["lib"].paged_store(s["pages"], s["batch"], s["q"].data_ptr(), s["q"].stride(0), s["q_out"].data_ptr(),
                         s["q_out"].stride(0), c["H"], s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(),
                         s["v"].stride(0), CODES[c["type"]], s["cos"].data_ptr(), s["sin"].data_ptr(), s["maxpos"],
                         st)
    return [s["q_out"], s["K"], s["V"]]


def _own_attn(s):
    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    s["lib"].paged_attn(s["pages"], s["batch"], s["q"].data_ptr(), CODES[c["type"]], c["H"] * c["hd"], c["H"],
                        c["hd"] ** -0.5, c["win"], c["sinks"], s["out"].data_ptr(), c["H"] * c["hd"],
                        s["lse"].data_ptr(), s["ws"].data_ptr(), s["ws_bytes"], st)
    return [s["out"], s["lse"]]


def _own_verify(s):
    c, x, st = s["case"], s["x"], torch.cuda.current_stream().cuda_stream
    y = s.get("y")
    s["lib"].spec_verify(x.data_ptr(), CODES[c["type"]], x.stride(0), 1.0 / c["temp"],
                         None if y is None else y.data_ptr(), 0 if y is None else y.stride(0),
                         1.0 / (c["dtemp"] or 1.0), s["N"], c["V"], s["row0"].data_ptr(), c["B"],
                         s["draft"].data_ptr(), s["u"].data_ptr(), s["noise"].data_ptr(), c["V"],
                         s["tokens"].data_ptr(), s["logp"].data_ptr(), s["accepted"].data_ptr(), s["ws"].data_ptr(),
                         s["ws_bytes"], st)
    return [s["tokens"], s["logp"], s["accepted"]]


def _rotate(x, pos, cos, sin):
    """RoPE of rows x [n][heads][hd]: the pairs (i, i + hd / 2) turned by their
    position's angles, in 32 bits."""
    a, b = x.float().chunk(2, 2)
    co, si = cos[pos][:, None], sin[pos][:, None]
    return torch.cat([a * co - b * si, b * co + a * si], 2)


def _plain_store(s):
    c, N, KV, hd, page = s["case"], s["N"], s["case"]["KV"], s["case"]["hd"], s["case"]["page"]
    i = torch.arange(N, device="cuda")
    b = torch.searchsorted(s["row0"][1:].long(), i, right=True)
    pos = s["len"].long()[b] - (s["row0"].long()[b + 1] - i)
    pg, off = s["table"].long()[b, pos // page], pos % page
    s["q_out"].copy_(_rotate(s["q"].reshape(N, c["H"], hd), pos, s["cos"], s["sin"]).reshape(N, -1))
    s["K"][pg, off] = _rotate(s["k"].reshape(N, KV, hd), pos, s["cos"], s["sin"]).to(s["K"].dtype)
    s["V"][pg, off] = s["v"].reshape(N, KV, hd).to(s["V"].dtype)
    return [s["q_out"], s["K"], s["V"]]


def _plain_attn(s):
    c, KV, hd = s["case"], s["case"]["KV"], s["case"]["hd"]
    G = c["H"] // KV
    out = torch.empty(s["N"], c["H"], hd, device="cuda", dtype=TYPES[c["type"]])
    lse = torch.empty(s["N"], c["H"], device="cuda")
    r = 0
    for b, (n, L) in enumerate(zip(s["rows"], s["lens"])):
        if n == 0:
            continue
        pg = s["table"][b, :-(-L // c["page"])].long()
        k = s["K"][pg].reshape(-1, KV, hd)[:L].float().permute(1, 2, 0).contiguous()
        v = s["V"][pg].reshape(-1, KV, hd)[:L].float().permute(1, 0, 2).contiguous()
        q = s["q"][r:r + n].float().reshape(n, KV, G, hd).permute(1, 0, 2, 3).reshape(KV, n * G, hd)
        t, p = torch.arange(L, device="cuda"), torch.arange(L - n, L, device="cuda")[:, None]
        hide = t > p
        if c["win"]:
            hide |= (t <= p - c["win"]) & (t >= c["sinks"])
        hide = hide.repeat_interleave(G, 0)
        step = KV if KV * n * G * L <= 1 << 29 else 1        # heads at once
        for h in range(0, KV, step):
            z = torch.matmul(q[h:h + step], k[h:h + step]).mul_(hd ** -0.5).masked_fill_(hide, -math.inf)
            m = z.amax(2, keepdim=True)
            z = z.sub_(m).exp_()
            tot = z.sum(2, keepdim=True)
            o = torch.matmul(z, v[h:h + step]).div_(tot)
            k2 = z.shape[0]
            out[r:r + n].view(n, KV, G, hd)[:, h:h + k2] = o.view(k2, n, G, hd).transpose(0, 1).to(out.dtype)
            lse[r:r + n].view(n, KV, G)[:, h:h + k2] = (m + tot.log()).view(k2, n, G).transpose(0, 1)
        r += n
    return [out, lse]


def _probs(x, scale):
    x = x.float()
    m = x.amax(1, keepdim=True)
    e = x.sub(m).mul_(scale).exp_()
    return e.div_(e.sum(1, keepdim=True))


def _plain_verify(s):
    c, B, V, N = s["case"], s["case"]["B"], s["case"]["V"], s["N"]
    first, last = s["row0"][:-1].long(), s["row0"][1:].long() - 1
    p = _probs(s["x"], 1.0 / c["temp"])
    i = torch.arange(N, device="cuda")
    d, drafted = s["draft"].long(), s["draft"] >= 0
    pd = p[i, d.clamp_min(0)]
    q = _probs(s["y"], 1.0 / c["dtemp"]) if c["dtemp"] else None
    qd = q[i, d.clamp_min(0)] if c["dtemp"] else torch.ones_like(pd)
    keep = drafted & (s["u"].double() * qd.double() < pd.double())
    seq = torch.searchsorted(s["row0"][1:].long(), i, right=True)
    # the first row of every sequence that keeps no draft
    stop = torch.full((B,), N, device="cuda").scatter_reduce_(0, seq, torch.where(keep, N, i), "amin")
    some = last >= first
    at = torch.where(some, stop, 0)
    w = p[at]
    if c["dtemp"]:
        left = (w - torch.where(drafted[at][:, None], q[at], 0.0)).clamp_min_(0.0)
        w = torch.where(left.sum(1, keepdim=True) > 0, left, w)
    else:
        w.scatter_(1, d[at].clamp_min(0)[:, None], torch.where(drafted[at], 0.0, w.gather(
            1, d[at].clamp_min(0)[:, None])[:, 0])[:, None])
    pick = (w / s["noise"]).argmax(1)
    tokens = torch.where(i < stop[seq], d, -1)
    logp = torch.where(i < stop[seq], pd.log(), 0.0)
    at = at[some]
    tokens[at] = pick[some]
    logp[at] = p[at, pick[some]].log()
    return [tokens.int(), logp, torch.where(some, stop - first, 0).int()]


_own = dict(store=_own_store, attn=_own_attn, verify=_own_verify)
_plain = dict(store=_plain_store, attn=_plain_attn, verify=_plain_verify)


# ------------------------------------------------------------------- work --
def work(case):
    """What a call cannot do without: rows in and out once; for attn the keys
    and values that some row of their sequence sees, and the products of every
    (row, head, visible token); for verify both models' rows, the exponentials
    of one row a sequence, and a few operations a logit."""
    c, (rows, lens) = case, _shape(case)
    N = sum(rows)
    if c["op"] == "verify":
        b, two = BYTES[c["type"]], 2 if c["dtemp"] else 1
        live = sum(n > 0 for n in rows)
        return dict(bytes=two * N * c["V"] * b + 4 * live * c["V"] + 16 * N, flops=4 * two * N * c["V"])
    tb, kb, hd = BYTES[c["type"]], BYTES[c["kv"]], c["hd"]
    if c["op"] == "store":
        return dict(bytes=N * hd * (2 * c["H"] * tb + 2 * c["KV"] * (tb + kb) + 4), flops=3 * N * (c["H"] + c["KV"]) * hd)
    pairs = seen = 0
    for n, L in zip(rows, lens):
        if n == 0:
            continue
        if not c["win"]:
            pairs += n * L - n * (n - 1) // 2
            seen += L
        else:
            lo = [max(0, p - c["win"] + 1) for p in range(L - n, L)]
            pairs += sum(p + 1 - a + min(a, c["sinks"]) for p, a in zip(range(L - n, L), lo))
            seen += L - lo[0] + min(lo[0], c["sinks"])
    return dict(bytes=2 * N * c["H"] * hd * tb + 4 * N * c["H"] + 2 * seen * c["KV"] * hd * kb,
                flops=4 * pairs * c["H"] * hd)


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    """What run returns, from the definitions in 64 bits."""
    return _exact[case["op"]](case, _inputs(case, seed))


def _exact_store(c, s):
    hd, page, H, KV = c["hd"], c["page"], c["H"], c["KV"]
    K, V = s["K"].double(), s["V"].double()
    q_out = torch.empty(s["N"], H * hd, device="cuda", dtype=torch.float64)
    table = s["table"].cpu().long()
    r = 0
    for b, (n, L) in enumerate(zip(s["rows"], s["lens"])):
        if n == 0:
            continue
        p = torch.arange(L - n, L)
        w = torch.complex(s["cos"][p.cuda()].double(), s["sin"][p.cuda()].double())[:, None]

        def turn(x, heads):              # each pair as a complex number
            x = x[r:r + n].double().reshape(n, heads, 2, hd // 2)
            z = torch.complex(x[:, :, 0], x[:, :, 1]) * w
            return torch.stack([z.real, z.imag], 2).reshape(n, heads, hd)
        q_out[r:r + n] = turn(s["q"], H).reshape(n, H * hd)
        pg, off = table[b][p // page].cuda(), (p % page).cuda()
        K[pg, off] = turn(s["k"], KV)
        V[pg, off] = s["v"][r:r + n].double().reshape(n, KV, hd)
        r += n
    return [q_out, K, V]


def _exact_attn(c, s):
    KV, hd, G = c["KV"], c["hd"], c["H"] // c["KV"]
    out = torch.zeros(s["N"], c["H"], hd, device="cuda", dtype=torch.float64)
    lse = torch.zeros(s["N"], c["H"], device="cuda", dtype=torch.float64)
    r = 0
    for b, (n, L) in enumerate(zip(s["rows"], s["lens"])):
        pg = s["table"][b, :-(-L // c["page"])].long()
        for h in range(KV if n else 0):
            k = s["K"][pg, :, h].reshape(-1, hd)[:L].double()
            v = s["V"][pg, :, h].reshape(-1, hd)[:L].double()
            for g in range(h * G, (h + 1) * G):
                for i in range(0, n, 1024):
                    m = min(1024, n - i)
                    p = torch.arange(L - n + i, L - n + i + m, device="cuda")[:, None]
                    t = torch.arange(L, device="cuda")[None, :]
                    see = t <= p
                    if c["win"]:
                        see = see & ((p - t < c["win"]) | (t < c["sinks"]))
                    z = (s["q"][r + i:r + i + m, g].double() @ k.T) / math.sqrt(hd)
                    z = torch.where(see, z, -math.inf)
                    l = torch.logsumexp(z, 1)
                    out[r + i:r + i + m, g] = torch.exp(z - l[:, None]) @ v
                    lse[r + i:r + i + m, g] = l
        r += n
    return [out, lse]


def _exact_verify(c, s):
    row0, draft, u = s["row0"].tolist(), s["draft"].tolist(), s["u"].tolist()
    tokens = torch.full((s["N"],), -1, dtype=torch.int32)
    logp, count = torch.zeros(s["N"], dtype=torch.float64), torch.zeros(c["B"], dtype=torch.int32)
    for b in range(c["B"]):
        lo, hi = row0[b], row0[b + 1]
        if lo == hi:
            continue
        lp = torch.log_softmax(s["x"][lo:hi].double() / c["temp"], 1)
        lq = torch.log_softmax(s["y"][lo:hi].double() / c["dtemp"], 1) if c["dtemp"] else None
        d = s["draft"][lo:hi].long().clamp_min(0)[:, None]
        lpd = lp.gather(1, d)[:, 0].tolist()
        lqd = lq.gather(1, d)[:, 0].tolist() if c["dtemp"] else [0.0] * (hi - lo)
        i = 0
        while draft[lo + i] >= 0 and u[lo + i] * math.exp(lqd[i]) < math.exp(lpd[i]):
            tokens[lo + i], logp[lo + i] = draft[lo + i], lpd[i]
            i += 1
        weight = lp[i].exp()
        if draft[lo + i] >= 0:
            if c["dtemp"]:
                weight = (weight - lq[i].exp()).clamp_min(0.0)
            else:
                weight[draft[lo + i]] = 0.0
        v = int((weight / s["noise"][b].double()).argmax())
        tokens[lo + i], logp[lo + i], count[b] = v, float(lp[i, v]), i
    return [tokens.cuda(), logp.cuda(), count.cuda()]


_exact = dict(store=_exact_store, attn=_exact_attn, verify=_exact_verify)
