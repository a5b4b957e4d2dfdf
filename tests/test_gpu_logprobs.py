"""tokenLogprobs against 64-bit results, Engine.score against the logits it does not bring back, and the
paged operators and the scores together as a serving host uses them."""
import numpy as np
import pytest

from batches import turned

pytestmark = pytest.mark.gpu


def dev(ctx, a):
    return ctx.from_numpy(np.ascontiguousarray(a))


def reference(x, targets, top):
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    e = np.exp(x - m)
    others = np.where(x == m, 0.0, e).sum(1) + ((x == m).sum(1) - 1.0)
    logz = np.log1p(others)
    lp = x - m - logz[:, None]
    ent = logz - (np.where(e > 0, (x - m), 0.0) * e).sum(1) / (1 + others)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return lp[np.arange(len(x)), targets], ent, ids, np.take_along_axis(lp, ids, 1)


def run(ctx, hip, x, targets, top, stride=None, offset=0):
    """x [n, V] laid out with `stride` elements a row, `offset` elements into its buffer; the rest is NaN."""
    n, V = x.shape
    stride = stride or V
    flat = np.full(offset + (n - 1) * stride + V, np.nan, np.float32)
    for r in range(n):
        flat[offset + r * stride:offset + r * stride + V] = x[r]
    b = dev(ctx, flat)
    outs = [dev(ctx, np.full(n + 1, 7.0, np.float32)), dev(ctx, np.full(n + 1, 7.0, np.float32)),
            dev(ctx, np.full(n * top + 1, 7, np.int32)), dev(ctx, np.full(n * top + 1, 7.0, np.float32))]
    views = [o.view(0, o.len - 4) for o in outs]
    hip.tokenLogprobs(ctx, hip.TokenLogprobsArgs(b.view(4 * offset, b.len - 4 * offset), dev(ctx, targets.astype(np.int32)), *views, n, V,
                                                 stride, top))
    got = [ctx.to_numpy(o, t) for o, t in zip(outs, (np.float32, np.float32, np.int32, np.float32))]
    assert all(g[-1] == 7 for g in got)  # nothing behind the outputs
    return got[0][:n], got[1][:n], got[2][:-1].reshape(n, top), got[3][:-1].reshape(n, top)


def tolerance(x):
    """exp's argument is rounded at |d| log2 e 2^-24 twice, which counts where the weight does (|d| e^d / Z
    at most 1, summed at most the entropy): 4 half steps per unit of it, the sums 48 more; x - m its own."""
    return 2.0 ** -24 * (64 + 4 * np.log(x.shape[1]) + 2 * np.abs(x[np.isfinite(x)]).max())


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 5, 5), (2, 33, 32), (1, 255, 7), (2, 256, 1), (1, 257, 0), (5, 2047, 20), (1, 2048, 20), (3, 2049, 32),
          (2, 8192, 5), (130, 8193, 3), (300, 1000, 20), (1, 16384, 1), (61, 16384, 0), (3, 30011, 32), (1, 65536, 20), (40, 65537, 5),
          (2, 600001, 32), (1, 2097152, 4)]


@pytest.mark.parametrize("n,V,top", SHAPES)
def test_token_logprobs(ctx, hip, n, V, top):
    print(f"[logprobs] n={n} V={V} top={top}", flush=True)
    g = np.random.default_rng([n, V])
    x = (g.standard_normal((n, V)) * 3).astype(np.float32)
    targets = np.where(g.random(n) < 0.5, g.integers(0, V, n), x.argmax(1))
    want = reference(x, targets, top)
    for stride, offset in ((V, 0), (V + 3, 1), (V + (-V) % 4 + 4, 4)):
        got = run(ctx, hip, x, targets, top, stride, offset)
        t = tolerance(x)
        assert np.all(np.abs(got[0] - want[0]) <= t) and np.all(np.abs(got[1] - want[1]) <= 2 * t * (1 + want[1]))
        assert np.array_equal(got[2], want[2]) and np.all(np.abs(got[3] - want[3]) <= t)


@pytest.mark.parametrize("V", [40, 5000, 70000])
def test_ties(ctx, hip, V):
    """Equal logits go to the lower id: rows of one value, of two values, and of both zeros."""
    g = np.random.default_rng(V)
    x = np.stack([np.zeros(V), g.integers(0, 2, V), np.where(g.random(V) < 0.5, 0.0, -0.0), g.integers(-3, 3, V), -np.arange(V) // 3]).astype(np.float32)
    got = run(ctx, hip, x, np.zeros(5, int), 32)
    want = reference(x, np.zeros(5, int), 32)
    assert np.array_equal(got[2], want[2])
    t = 2.0 ** -24 * (64 + 4 * np.log(V) + 64)
    assert np.all(np.abs(got[0] - want[0]) <= t) and np.all(np.abs(got[3] - want[3]) <= t * (1 + np.abs(want[3])))


@pytest.mark.parametrize("V", [100, 30000])
def test_masked_and_undefined(ctx, hip, V):
    g = np.random.default_rng(V)
    x = g.standard_normal((9, V)).astype(np.float32)
    x[0, 3:] = -np.inf                        # three tokens are left
    x[1, :] = -np.inf
    x[1, V - 1] = 2.0                         # one is
    x[2, :] = -np.inf                         # none
    x[3, V // 2] = np.nan
    x[4, V // 3] = np.inf
    x[5, ::2] = np.finfo(np.float32).min      # the type's lowest value as a mask
    x[6, :] = np.finfo(np.float32).min
    x[7] *= 1e30
    targets = np.array([1, V - 1, 0, 0, 0, 1, 0, int(x[7].argmax()), -1])
    lp, ent, ids, tops = run(ctx, hip, x, targets, 5)
    for r in (2, 3, 4):
        assert np.isnan([lp[r], ent[r], *tops[r]]).all() and np.all(ids[r] == -1)
    assert np.isnan(lp[8]) and np.isfinite(ent[8])  # no such target; the row is whole
    with np.errstate(invalid="ignore"):
        want = reference(x, np.maximum(targets, 0), 5)
    ok = [0, 1, 5, 6, 7, 8]
    assert np.array_equal(ids[ok], want[2][ok])
    assert np.all(np.abs(ent[ok] - want[1][ok]) <= 1e-5 * (1 + want[1][ok]))
    assert np.all(np.abs(lp[ok[:5]] - want[0][ok[:5]]) <= 1e-5 * (1 + np.abs(want[0][ok[:5]])))
    fin = np.isfinite(want[3][ok])
    assert np.array_equal(fin, np.isfinite(tops[ok])) and np.all(tops[ok][~fin] == -np.inf)
    assert np.all(np.abs(tops[ok][fin] - want[3][ok][fin]) <= 1e-5 * (1 + np.abs(want[3][ok][fin])))
    assert lp[1] == 0.0 and ent[1] == 0.0
    for t in (2 ** 31 - 1, -2 ** 31, V):
        assert np.isnan(run(ctx, hip, x[:1], np.array([t]), 1)[0][0])


def test_almost_certain(ctx, hip):
    """The likely token's log probability and the entropy keep their relative accuracy: the sums of the
    others hold 2^-17 of themselves (arguments of up to 40 rounded at 2^-23)."""
    V = 20000
    x = (np.random.default_rng(3).standard_normal((4, V)) * 0.5).astype(np.float32)
    for r, up in enumerate((12, 18, 25, 40)):
        x[r, 777 + r] = up
    targets = 777 + np.arange(4)
    lp, ent, _, _ = run(ctx, hip, x, targets, 0)
    want = reference(x, targets, 1)
    assert np.all(np.abs(lp / want[0] - 1) <= 2.0 ** -17) and np.all(np.abs(ent / want[1] - 1) <= 2.0 ** -17)


def test_parts_of_the_outputs(ctx, hip):
    x = np.random.default_rng(4).standard_normal((3, 9000)).astype(np.float32)
    targets = np.array([5, 6, 7], np.int32)
    whole = run(ctx, hip, x, targets, 4)
    xb, tb, none = dev(ctx, x), dev(ctx, targets), hip.Buf()
    for take in range(1, 8):
        outs = [ctx.createBuffer(b) if take >> i & 1 else none for i, b in enumerate((12, 12, 48))]
        tops = ctx.createBuffer(48) if take & 4 else none
        hip.tokenLogprobs(ctx, hip.TokenLogprobsArgs(xb, tb if take & 1 else none, *outs, tops, 3, 9000, 9000, 4 if take & 4 else 0))
        for i, t in enumerate((np.float32, np.float32, np.int32)):
            if take >> i & 1:
                assert np.array_equal(ctx.to_numpy(outs[i], t), whole[i].ravel())


def test_logprobs_graph(ctx, hip):
    n, V, top = 7, 20000, 9
    g = np.random.default_rng(5)
    x = g.standard_normal((4, n, V)).astype(np.float32)
    xb, tb = dev(ctx, x[0]), dev(ctx, g.integers(0, V, n).astype(np.int32))
    outs = [ctx.createBuffer(n * 4) for _ in range(2)] + [ctx.createBuffer(n * top * 4) for _ in range(2)]
    args = hip.TokenLogprobsArgs(xb, tb, *outs, n, V, V, top)
    hip.tokenLogprobs(ctx, args)
    graph = ctx.capture(lambda: hip.tokenLogprobs(ctx, args))
    for i in range(4):
        ctx.upload(xb, 0, x[i])
        hip.tokenLogprobs(ctx, args)
        eager = [ctx.to_numpy(o, np.uint32) for o in outs]
        for o in outs:
            ctx.zero(o, o.len)
        graph.launch()
        assert all(np.array_equal(ctx.to_numpy(o, np.uint32), e) for o, e in zip(outs, eager))
    graph.destroy()


@pytest.mark.parametrize("fused", [False, True])
def test_engine_score(ctx, hip, fused):
    import synth_model
    from qw3_amd import engine as E
    cfg, tensors = synth_model.load()[:2]
    w = E.Weights(ctx, tensors, cfg)
    vocab = w.cfg["vocab_size"]
    toks = [(7 * i + 3) % vocab for i in range(20)]
    a, b = (E.Engine(ctx, w, 32, 64, hip.DTYPE_F16, fused) for _ in range(2))
    for part, top in ((toks[:13], 5), (toks[13:14], 1), (toks[14:], 0)):
        targets = [(3 * t + 1) % vocab for t in part]
        logits = a.forward(part)
        got = b.score(part, targets, top)
        want = reference(logits, np.array(targets), top)
        t = tolerance(logits)
        assert np.all(np.abs(got["logprobs"] - want[0]) <= t) and np.all(np.abs(got["entropy"] - want[1]) <= 2 * t * (1 + want[1]))
        assert np.array_equal(got["top_ids"], want[2]) and np.all(np.abs(got["top_logprobs"] - want[3]) <= t)
    assert a.pos == b.pos == 20


def test_a_served_batch(ctx, hip):
    """Prompts of three lengths admitted at once, then decode steps: projections, pagedAppend, pagedAttention,
    the head and tokenLogprobs, the last steps with pagedDecode over the same pool; every sequence's log
    probabilities against the same layer over its own contiguous cache in 64 bits."""
    g = np.random.default_rng(9)
    hid, hq, hkv, d, V, page = 256, 8, 2, 64, 3001, 16
    prompts, steps = [37, 5, 130], 5
    norm = lambda *s: g.standard_normal(s).astype(np.float32)  # noqa: E731
    wq, wk, wv, wo, head = (norm(n, k) / np.float32(k ** 0.5) for n, k in ((hq * d, hid), (hkv * d, hid), (hkv * d, hid), (hid, hq * d), (V, hid)))
    qn, kn = (g.normal(1, 0.02, d).astype(np.float32) for _ in range(2))
    total = [n + steps for n in prompts]
    x = [norm(n, hid) for n in total]
    nxt = [g.integers(0, V, n) for n in total]
    most = max(-(-n // page) for n in total)
    table = g.permutation(3 * most).astype(np.int32).reshape(3, most)
    scale = float(np.float32(d ** -0.5))
    F = hip.DTYPE_F32
    W = {n: dev(ctx, a) for n, a in dict(q=wq, k=wk, v=wv, o=wo, h=head, qn=qn, kn=kn).items()}
    kp, vp = (ctx.createBuffer(hkv * 3 * most * page * d * 2) for _ in range(2))
    tb = dev(ctx, table)

    def step(rows, lens, targets, decode):
        T = sum(map(len, rows))
        xb = dev(ctx, np.concatenate(rows))
        q, k, v, attn, hb, lg = (ctx.createBuffer(T * n * 4) for n in (hq * d, hkv * d, hkv * d, hq * d, hid, V))
        hip.matmulGroup(ctx, hip.MatmulGroupArgs.of(xb, F, T, hid, [(W["q"], q, hq * d), (W["k"], k, hkv * d), (W["v"], v, hkv * d)]))
        sl = dev(ctx, np.array(lens, np.int32))
        if decode:
            hip.pagedDecode(ctx, hip.PagedDecodeArgs(q, k, v, W["qn"], W["kn"], kp, vp, tb, sl, attn, 3, hq, hkv, d, page, 3 * most, most,
                                                     max(lens), 1e-6, 1e6, 1.0, scale))
        else:
            st = dev(ctx, np.concatenate([[0], np.cumsum([len(r) for r in rows])]).astype(np.int32))
            shape = (F, T, 3, hq, hkv, d, page, 3 * most, most, max(lens))
            hip.pagedAppend(ctx, hip.PagedAppendArgs(q, k, v, W["qn"], W["kn"], q, kp, vp, tb, st, sl, *shape, 1e-6, 1e6, 1.0))
            hip.pagedAttention(ctx, hip.PagedAttentionArgs(q, kp, vp, tb, st, sl, attn, *shape, scale))
        hip.matmulAdd(ctx, hip.MatmulAddArgs(attn, W["o"], F, xb, hb, T, hid, hq * d))
        hip.matmul(ctx, hip.MatmulArgs(hb, W["h"], F, lg, T, V, hid))
        lp = ctx.createBuffer(T * 4)
        hip.tokenLogprobs(ctx, hip.TokenLogprobsArgs(lg, dev(ctx, np.concatenate(targets).astype(np.int32)), lp, hip.Buf(), hip.Buf(), hip.Buf(),
                                                     T, V, V, 0))
        return np.split(ctx.to_numpy(lp, np.float32), np.cumsum([len(r) for r in rows])[:-1])

    got = [[] for _ in prompts]
    for i in range(steps + 1):
        span = [slice(0, n) if i == 0 else slice(n + i - 1, n + i) for n in prompts]
        for b, v in enumerate(step([x[b][span[b]] for b in range(3)], [n + i for n in prompts], [nxt[b][span[b]] for b in range(3)], i >= 3)):
            got[b].append(v)
    for b, n in enumerate(total):
        x64, pos = x[b].astype(np.float64), np.arange(n)
        q = turned((x64 @ wq.T.astype(np.float64)).reshape(n, hq, d), qn, pos, 1e6, 1e-6)
        k = turned((x64 @ wk.T.astype(np.float64)).reshape(n, hkv, d), kn, pos, 1e6, 1e-6).astype(np.float16).astype(np.float64)
        v = (x64 @ wv.T.astype(np.float64)).reshape(n, hkv, d).astype(np.float16).astype(np.float64)
        o = np.empty((n, hq, d))
        for h in range(hq):
            s = q[:, h] @ k[:, h // (hq // hkv)].T * scale
            s[pos[None] > pos[:, None]] = -np.inf
            w = np.exp(s - s.max(1, keepdims=True))
            o[:, h] = w @ v[:, h // (hq // hkv)] / w.sum(1, keepdims=True)
        lg = (x64 + o.reshape(n, -1) @ wo.T) @ head.T.astype(np.float64)
        want = (lg - lg.max(1, keepdims=True) - np.log(np.exp(lg - lg.max(1, keepdims=True)).sum(1, keepdims=True)))[pos, nxt[b]]
        # k and v rows may round to either side of a step of f16 (2^-11 of them) where f32 and f64 projections part:
        # a rare element, 2^-11 of it through softmax and two projections of unit gain
        assert np.all(np.abs(np.concatenate(got[b]) - want) <= 2e-3), b


@pytest.mark.parametrize("V,at", [(8193, 8192), (2 ** 19 + 1, 2 ** 19), (70001, 70000), (300, 299)])
@pytest.mark.parametrize("rest", [0.0, -np.inf])
def test_nan_alone_in_a_segment(ctx, hip, V, at, rest):
    """A NaN whose part of the row holds nothing else, or nothing else but -inf, undoes the row all the same."""
    x = np.random.default_rng(V).standard_normal((2, V)).astype(np.float32)
    x[1, V // 8192 * 8192:] = rest
    x[1, at] = np.nan
    lp, ent, ids, tops = run(ctx, hip, x, np.zeros(2, int), 3)
    assert np.isfinite([lp[0], ent[0], *tops[0]]).all()
    assert np.isnan([lp[1], ent[1], *tops[1]]).all() and np.all(ids[1] == -1)


def test_two_graphs_share_the_workspaces(ctx, hip):
    """Attention and scores of two shapes, each in a graph of its own, replayed in turn with eager calls that outgrow
    the workspace between them: every replay as the eager calls, bit for bit."""
    from batches import Batch
    calls = []
    for seed, lens, new, n, V in ((1, [5000, 900], [1, 70], 40, 70001), (2, [12000], [1], 3, 300000)):
        c = Batch(seed, lens, new, 16, 2, 128)
        out, bufs = ctx.createBuffer(c.rows * c.hq * c.d * 4), [dev(ctx, a) for a in (c.q, c.kp, c.vp, c.table, c.starts, c.seq_lens)]
        at = hip.PagedAttentionArgs(*bufs, out, *c.shape(hip, False), c.scale)
        x = dev(ctx, c.g.standard_normal((n, V)).astype(np.float32))
        outs = [ctx.createBuffer(n * 4) for _ in range(2)] + [ctx.createBuffer(n * 20 * 4) for _ in range(2)]
        lp = hip.TokenLogprobsArgs(x, dev(ctx, c.g.integers(0, V, n).astype(np.int32)), *outs, n, V, V, 20)

        def both(at=at, lp=lp):
            hip.pagedAttention(ctx, at)
            hip.tokenLogprobs(ctx, lp)

        both()
        got = [ctx.to_numpy(o, np.uint32) for o in (out, *outs)]
        calls.append((both, ctx.capture(both), (out, *outs), got))
    big = ctx.createBuffer(8000 * 20000 * 4)  # 6.6 MB of states and keys, more than a workspace begins with
    ctx.zero(big, big.len)
    tops = [ctx.createBuffer(8000 * 32 * 4) for _ in range(2)]
    none = hip.Buf()
    for i in range(4):
        for both, graph, outs, want in calls:
            for o in outs:
                ctx.zero(o, o.len)
            graph.launch()
            assert all(np.array_equal(ctx.to_numpy(o, np.uint32), w) for o, w in zip(outs, want))
            if i == 1:
                hip.tokenLogprobs(ctx, hip.TokenLogprobsArgs(big, none, none, none, *tops, 8000, 20000, 20000, 32))
                assert np.array_equal(ctx.to_numpy(tops[0], np.int32), np.tile(np.arange(32), 8000))
                both()
    for _, graph, _, _ in calls:
        graph.destroy()


def part_lengths(top, aligned):
    """Lengths of a part of a row around those where top to 1.5 top of its threads hold a logit (four each where
    the rows are 16-byte aligned)."""
    k = 4 if aligned else 1
    return sorted({n for n in (k * top - k, k * top - k + 1, k * top, k * (top + 1), k * (top + top // 2), k * (top + top // 2) + 1) if n >= top})


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("top", [2, 5, 20, 32])
@pytest.mark.parametrize("segs", [0, 5])
def test_few_finite_logits_in_a_part(ctx, hip, segs, top, aligned):
    """A mask that leaves fewer finite logits than alternatives, in a short row and in the short last part of a long
    one (2048 logits a part where rows of more than 8192 are few): every finite one is among the alternatives, then the lowest ids."""
    for last in part_lengths(top, aligned):
        V = 2048 * segs + last
        g = np.random.default_rng([segs, top, last])
        for left in sorted({1, top // 2, top - 1} - {0}):
            x = np.full((3, V), -np.inf, np.float32)
            for r in range(3):
                x[r, 2048 * segs + g.choice(last, left, replace=False)] = g.standard_normal(left) * 3
            if segs:
                x[1, :2048 * segs] = g.standard_normal(2048 * segs) - 20  # less likely ones in the parts before
                x[2, g.choice(2048 * segs, top, replace=False)] = 30 + g.standard_normal(top)  # and likelier ones
            targets = x.argmax(1)
            with np.errstate(invalid="ignore"):
                want = reference(x, targets, top)
            stride = V + (-V) % 4 if aligned else V + 1 - V % 2
            got = run(ctx, hip, x, targets, top, stride)
            assert np.array_equal(got[2], want[2]), (V, left)
            t, finite = tolerance(x), np.isfinite(want[3])
            assert np.array_equal(np.isfinite(got[3]), finite) and np.all(got[3][~finite] == -np.inf)
            assert np.all(np.abs(got[3][finite] - want[3][finite]) <= t)
            assert np.all(np.abs(got[0] - want[0]) <= t) and np.all(np.abs(got[1] - want[1]) <= 2 * t * (1 + want[1]))
