"""The operators of a paged batch and of scored tokens, as a serving host of the engine calls them: new rows appended to a
paged pool with their norm and rotation (`pagedAppend`), attention of each sequence's new tokens over that pool
(`pagedAttention`), and the log probabilities of given tokens with entropy and top alternatives (`tokenLogprobs`).

Shapes: the 32 q / 4 kv and 64 q / 4 kv heads of 128 of Qwen3-30B-A3B and Qwen3-235B-A22B, the 16 / 2 heads of 64 of the tests,
vocabularies of the tests' size, of the benchmarks' models and generic ones.

A batch (`op` append or attention) has `seqs` sequences with ctx_lo .. ctx_hi tokens cached; the first `chunks` of them
bring new_lo .. new_hi new tokens, the others one. `own` false computes the operators in plain torch, true calls them: on the
context's stream, which torch's does not wait for, so that a synchronization goes before anything that reads what they wrote.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e6
DEV = "cuda"


def _batch(name, op, seqs, ctx, chunks=0, new=(1, 1), heads=(32, 4, 128), page=16, q="f32"):
    return dict(name=name, op=op, seqs=seqs, ctx_lo=ctx[0], ctx_hi=ctx[1], chunks=chunks, new_lo=new[0], new_hi=new[1],
                hq=heads[0], hkv=heads[1], d=heads[2], page=page, q=q)


def listed():
    return [
        # a chat's next token: the smallest append, latency alone
        _batch("append, one token", "append", 1, (4095, 4095)),
        # a decode step of a serving batch with wide heads
        _batch("append, 32 sequences", "append", 32, (512, 4000), heads=(64, 4, 128), q="f16"),
        # prompts of every length admitted together
        _batch("append, ragged prompts", "append", 9, (0, 700), 9, (3, 900), q="f16", page=32),
        # a chat's next token late in an 8K context
        _batch("attention, one token at 8K", "attention", 1, (8191, 8191)),
        # a serving batch: sequences of very different lengths
        _batch("attention, 32 sequences", "attention", 32, (511, 16383)),
        # a few tokens each, as drafted tokens are verified; heads of 64, pages of 48
        _batch("attention, 5 tokens x 8", "attention", 8, (100, 3000), 8, (5, 5), heads=(16, 2, 64), page=48),
        # a long prompt, q as 16-bit rows
        _batch("attention, prompt of 2048", "attention", 1, (0, 0), 1, (2048, 2048), q="f16"),
        # the next user turn of a long chat: a ragged chunk after 6000 cached tokens, wide heads
        _batch("attention, 203 at 6000", "attention", 1, (6000, 6000), 1, (203, 203), heads=(64, 4, 128)),
        # continuous batching: two prompts among 22 decoding sequences
        _batch("attention, mixed batch", "attention", 24, (64, 4000), 2, (100, 500)),
        # a sampled token's probability with its alternatives
        dict(name="logprobs, one row", op="logprobs", rows=1, vocab=65536, top=20, pad=0),
        # a short prompt's probabilities: no alternatives
        dict(name="logprobs, 61 rows", op="logprobs", rows=61, vocab=16384, top=0, pad=0),
        # texts scored in bulk
        dict(name="logprobs, 512 rows", op="logprobs", rows=512, vocab=65536, top=5, pad=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "logprobs"])
    if op == "logprobs":
        vocab = _log_int(rng, 300, 131072)
        return dict(op=op, rows=_log_int(rng, 1, max(2, min(3000, 16000000 // vocab))), vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]),
                    pad=rng.choice([0, 0, 1, 64]))
    heads = rng.choice([(32, 4, 128), (32, 4, 128), (64, 4, 128), (16, 2, 64), (8, 8, 128), (20, 4, 64)])
    seqs = _log_int(rng, 1, 32)
    chunks = rng.choice([0, 0, 1, seqs])
    hi = max(2, min(_log_int(rng, 2, 1500), 1500 // max(1, chunks)))
    # no dearer than the listed ones: bytes of the caches; products of the rows that see a position, and of all (the plain form)
    hq, hkv, d = heads
    most = min(4e8 / (seqs * hkv * d * 4), 3.5e10 / (4 * d * hq * (seqs + chunks * hi)), 4e8 / (hq * (seqs + chunks * hi) * seqs))
    ctx_hi = int(max(1, min(_log_int(rng, 1, 12000), most - hi)))
    c = _batch("", op, seqs, (rng.randint(0, ctx_hi), ctx_hi), chunks, (rng.randint(1, hi), hi), heads,
               rng.choice([16, 16, 32, 48]), rng.choice(["f32", "f16"]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _sizes(c):
    """Every sequence's cached and new tokens: a fixed spread over the case's ranges."""
    g = random.Random(c["seqs"] * 1000003 + c["ctx_hi"] * 101 + c["new_hi"])
    ctx = [g.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["seqs"])]
    new = [g.randint(c["new_lo"], c["new_hi"]) if b < c["chunks"] else 1 for b in range(c["seqs"])]
    return ctx, new


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device=DEV) * std + mean

    if c["op"] == "logprobs":
        n, V, top = c["rows"], c["vocab"], c["top"]
        x = torch.empty(n, V + c["pad"], device=DEV)
        x.copy_(normal(n, V + c["pad"], std=2.5))
        f = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
        # a text's own tokens are likelier than chance: half of them among the larger logits
        targets = torch.randint(0, V, (n,), generator=g, device=DEV)
        targets[::2] = x[::2, :V].argmax(1)
        s = dict(c=dict(c), x=x, targets=targets.to(torch.int32), logprobs=f(n), entropy=f(n),
                 top_ids=torch.zeros(n, top, dtype=torch.int32, device=DEV), top_logprobs=f(n, top))
        torch.cuda.synchronize()  # the inputs are made on torch's stream, the calls run on the context's
        return s
    ctx, new = _sizes(c)
    lens = [a + b for a, b in zip(ctx, new)]
    pages = [-(-n // c["page"]) for n in lens]
    n_pages, most = sum(pages), max(pages)
    perm = np.random.default_rng([seed, n_pages]).permutation(n_pages).astype(np.int32)  # pages handed out in any order
    table, at = np.full((c["seqs"], most), -1, np.int32), 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    hq, hkv, d, T = c["hq"], c["hkv"], c["d"], sum(new)
    qt = torch.float16 if c["q"] == "f16" else torch.float32
    s = dict(c=dict(c), ctx=ctx, new=new, lens=lens, T=T, n_pages=n_pages, max_len=max(lens),
             table=torch.from_numpy(table).to(DEV), starts=_i32([0] + np.cumsum(new).tolist()), seq_lens=_i32(lens),
             k_pool=normal(hkv, n_pages * c["page"], d).half(), v_pool=normal(hkv, n_pages * c["page"], d).half())
    if c["op"] == "append":
        s |= dict(q=normal(T, hq, d), k=normal(T, hkv, d), v=normal(T, hkv, d), q_norm=normal(d, std=0.02, mean=1.0),
                  k_norm=normal(d, std=0.02, mean=1.0), q_out=torch.zeros(T, hq, d, dtype=qt, device=DEV))
    else:
        s |= dict(q=normal(T, hq, d).to(qt), out=torch.zeros(T, hq * d, device=DEV))
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _rows(s):
    """Sequence and position of every new row."""
    new = torch.tensor(s["new"], device=DEV)
    b = torch.repeat_interleave(torch.arange(len(s["new"]), device=DEV), new, output_size=s["T"])
    return b, s["seq_lens"].long()[b] - new[b] + torch.arange(s["T"], device=DEV) - s["starts"].long()[b]


def _slots(s, b, pos):
    page = s["c"]["page"]
    return s["table"][b, pos // page].long() * page + pos % page


def _turned(x, w, pos):
    """Norm over the head, then the rotation of element i with element i + d / 2; angles in 64 bits."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    h = x.shape[-1] // 2
    inv = THETA ** (-torch.arange(h, dtype=torch.float64, device=DEV) / h)
    a = pos.double()[:, None] * inv
    co, si = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    u, v = x[..., :h], x[..., h:]
    return torch.cat([u * co - v * si, u * si + v * co], -1)


def _plain_append(s):
    b, pos = _rows(s)
    slot = _slots(s, b, pos)
    s["k_pool"][:, slot] = _turned(s["k"], s["k_norm"], pos).half().transpose(0, 1)
    s["v_pool"][:, slot] = s["v"].half().transpose(0, 1)
    return dict(q=_turned(s["q"], s["q_norm"], pos).to(s["q_out"].dtype), k_pool=s["k_pool"], v_pool=s["v_pool"])


def _plain_attention(s):
    """A score for every new row and every cached position of the batch, masked where the row doesn't see the position."""
    c = s["c"]
    b, pos = _rows(s)
    lens = s["seq_lens"].long()
    kb = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), lens, output_size=sum(s["lens"]))
    kp = torch.arange(sum(s["lens"]), device=DEV) - (torch.cumsum(lens, 0) - lens)[kb]
    slot = _slots(s, kb, kp)
    k, v = s["k_pool"][:, slot].float(), s["v_pool"][:, slot].float()
    hq, hkv, d, T = c["hq"], c["hkv"], c["d"], s["T"]
    G = hq // hkv
    q = s["q"].float().view(T, hkv, G, d).permute(1, 2, 0, 3).reshape(hkv, G * T, d)
    x = (q @ k.transpose(1, 2).contiguous()).view(hkv, G, T, -1) * d ** -0.5
    x.masked_fill_(~((kb[None] == b[:, None]) & (kp[None] <= pos[:, None])), -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    o = (x.view(hkv, G * T, -1) @ v) / x.view(hkv, G * T, -1).sum(-1, keepdim=True)
    return o.view(hkv, G, T, d).permute(2, 0, 1, 3).reshape(T, hq * d)


def _plain_logprobs(s):
    c = s["c"]
    x = s["x"][:, :c["vocab"]]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True, dtype=torch.float64)
    lp = ((x - m).double() - torch.log(z)).float()
    r = dict(logprobs=lp.gather(1, s["targets"].long()[:, None])[:, 0], entropy=-((e / z) * lp).sum(1, dtype=torch.float64).float())
    if c["top"]:
        _, i = torch.sort(x, dim=1, descending=True, stable=True)
        i = i[:, :c["top"]]
        r |= dict(top_ids=i.to(torch.int32), top_logprobs=lp.gather(1, i))
    return r


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
_ctx = None


def _buf(H, t):
    """A view of a device tensor as the C ABI takes it."""
    return H.Buf(t.data_ptr(), 0, t.numel() * t.element_size())


def _own(s):
    """The call on a state's buffers; its arguments are made once, as a host that calls it step after step keeps them."""
    import qw3_amd.hip as H
    global _ctx
    if _ctx is None:
        _ctx = H.Ctx.init(0)
    c, op = s["c"], s["c"]["op"]
    if "args" not in s:
        B = lambda *names: [_buf(H, s[n]) for n in names]  # noqa: E731
        if op == "logprobs":
            s["args"] = H.TokenLogprobsArgs(*B("x", "targets", "logprobs", "entropy", "top_ids", "top_logprobs"), c["rows"], c["vocab"],
                                            c["vocab"] + c["pad"], c["top"])
        else:
            dt = H.DTYPE_F16 if c["q"] == "f16" else H.DTYPE_F32
            shape = (dt, s["T"], c["seqs"], c["hq"], c["hkv"], c["d"], c["page"], s["n_pages"], s["table"].shape[1], s["max_len"])
            if op == "append":
                s["args"] = H.PagedAppendArgs(*B("q", "k", "v", "q_norm", "k_norm", "q_out", "k_pool", "v_pool", "table", "starts", "seq_lens"),
                                              *shape, EPS, THETA, 1.0)
            else:
                s["args"] = H.PagedAttentionArgs(*B("q", "k_pool", "v_pool", "table", "starts", "seq_lens", "out"), *shape, c["d"] ** -0.5)
    if op == "logprobs":
        H.tokenLogprobs(_ctx, s["args"])
        return {n: s[n] for n in ("logprobs", "entropy") + (("top_ids", "top_logprobs") if c["top"] else ())}
    if op == "append":
        H.pagedAppend(_ctx, s["args"])
        return dict(q=s["q_out"], k_pool=s["k_pool"], v_pool=s["v_pool"])
    H.pagedAttention(_ctx, s["args"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}[state["c"]["op"]](state)


# ---------------------------------------------------------------------------
# work and the 64-bit results
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return dict(bytes=4 * n + c["rows"] * (12 + 8 * c["top"]), flops=6 * n)
    ctx, new = _sizes(c)
    hq, hkv, d, T = c["hq"], c["hkv"], c["d"], sum(new)
    qb = 2 if c["q"] == "f16" else 4
    tables = 4 * (2 * c["seqs"] + 1)
    if c["op"] == "append":
        return dict(bytes=T * d * (hq * (4 + qb) + hkv * 12) + 8 * d + 4 * T + tables, flops=T * d * 8 * (hq + hkv))
    L = sum(ctx) + T
    seen = sum(n * a + n * (n + 1) // 2 for a, n in zip(ctx, new))
    return dict(bytes=4 * L * hkv * d + T * hq * d * (qb + 4) + 4 * L / c["page"] + tables, flops=4 * d * hq * seen)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "logprobs":
        x = s["x"][:, :c["vocab"]].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        r = dict(logprobs=lp[torch.arange(c["rows"], device=DEV), s["targets"].long()], entropy=-(lp.exp() * lp).sum(1))
        if c["top"]:
            ids = torch.argsort(-x, dim=1, stable=True)[:, :c["top"]]
            r |= dict(top_ids=ids.to(torch.int32), top_logprobs=torch.take_along_dim(lp, ids, 1))
        return r
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    kp, vp = s["k_pool"].double(), s["v_pool"].double()
    out, at = torch.empty(s["T"], hq, d, dtype=torch.float64, device=DEV), 0
    for b, (n0, n) in enumerate(zip(s["ctx"], s["new"])):
        p = torch.arange(n0 + n, device=DEV)
        slots = s["table"][b].long()[p // page] * page + p % page
        if c["op"] == "append":
            ang = torch.outer(p[n0:].double(), torch.pow(torch.tensor(THETA, dtype=torch.float64, device=DEV),
                                                         -2.0 * torch.arange(d // 2, dtype=torch.float64, device=DEV) / d))
            z = torch.polar(torch.ones_like(ang), ang)[:, None]

            def turn(x, w):
                x = x.double()
                x = x / x.square().mean(-1, keepdim=True).add(EPS).sqrt() * w.double()
                y = torch.complex(x[..., :d // 2], x[..., d // 2:]) * z
                return torch.cat([y.real, y.imag], -1)

            out[at:at + n] = turn(s["q"][at:at + n], s["q_norm"])
            kp[:, slots[n0:]] = turn(s["k"][at:at + n], s["k_norm"]).transpose(0, 1)
            vp[:, slots[n0:]] = s["v"][at:at + n].double().transpose(0, 1)
        else:
            hidden = p[None] > p[n0:, None]
            for h in range(hq):
                kv = h // (hq // hkv)
                w = torch.softmax((s["q"][at:at + n, h].double() @ kp[kv, slots].T / math.sqrt(d)).masked_fill(hidden, -math.inf), 1)
                out[at:at + n, h] = w @ vp[kv, slots]
        at += n
    return dict(q=out, k_pool=kp, v_pool=vp) if c["op"] == "append" else out.view(s["T"], hq * d)
