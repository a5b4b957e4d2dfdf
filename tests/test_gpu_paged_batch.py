"""pagedAppend and pagedAttention against 64-bit results: lengths from one token to long ones, pages that
end inside a tile, group sizes and head sizes, rows behind the last sequence, sequences without rows, NaN
where nothing looks, device-side entries out of range, and both in a captured graph."""
import numpy as np
import pytest

from batches import Batch, turned

pytestmark = pytest.mark.gpu
EPS, THETA = 1e-6, 1e6


def dev(ctx, a):
    return ctx.from_numpy(np.ascontiguousarray(a))


def run_attention(ctx, hip, c, q_f16=False, fill=7.0, scale=None, **kw):
    out = dev(ctx, np.full((c.rows, c.hq * c.d), fill, np.float32))
    args = hip.PagedAttentionArgs(dev(ctx, c.q), dev(ctx, c.kp), dev(ctx, c.vp), dev(ctx, c.table), dev(ctx, c.starts), dev(ctx, c.seq_lens),
                                  out, *c.shape(hip, q_f16), c.scale if scale is None else scale)
    for k, v in kw.items():
        setattr(args, k, v)
    hip.pagedAttention(ctx, args)
    got = ctx.to_numpy(out, np.float32, (c.rows, c.hq, c.d))
    hip.pagedAttention(ctx, args)
    again = ctx.to_numpy(out, np.float32, (c.rows, c.hq, c.d))
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32))  # the same bits every time
    return got


def check_attention(ctx, hip, c, q_f16=False):
    want, tol = c.attention()
    got = run_attention(ctx, hip, c, q_f16)
    assert np.all(got[c.T:] == 7.0)  # rows that no sequence holds
    err = np.abs(got[:c.T] - want[:c.T])
    assert np.all(err <= tol[:c.T]), (float((err / tol[:c.T]).max()), np.unravel_index(np.argmax(err / tol[:c.T]), err.shape))
    # and on the whole 1e-5, where the scores allow it: one of size s in f32 is rounded by s 2^-24 in its sum and
    # again in its scaling, which moves its weight, and so the output, by as much of itself, the weights' sum too
    d = got[:c.T] - want[:c.T]
    if c.T:
        assert np.linalg.norm(d) <= (1e-5 + 4 * c.largest * 2.0 ** -24) * np.linalg.norm(want[:c.T])


ATTENTION = [  # ctx, new, hq, hkv, d, page
    ([0], [1], 32, 4, 128, 16),               # one token, one position
    ([14], [1], 32, 4, 128, 16),
    ([15], [1], 32, 4, 128, 16),              # the last slot of a page
    ([16], [1], 4, 4, 64, 16),
    ([63, 64, 65], [1, 1, 1], 8, 2, 64, 16),
    ([127, 128, 129, 255, 256, 257], [1] * 6, 32, 4, 128, 32),
    ([1000], [1], 64, 4, 128, 48),
    ([8191], [1], 32, 4, 128, 16),            # a long cache split over workgroups
    ([8190, 3, 100], [1, 1, 1], 5, 1, 128, 16),
    ([20000], [1], 8, 1, 64, 64),
    ([0], [2], 32, 4, 128, 16),
    ([0], [16], 8, 1, 128, 16),
    ([0], [17], 8, 1, 128, 16),
    ([5], [4], 32, 4, 128, 16),               # 32 query rows of a kv head
    ([5], [5], 32, 4, 128, 16),               # 40
    ([0], [128], 2, 2, 64, 16),
    ([0], [129], 2, 2, 64, 48),
    ([31], [300], 6, 2, 128, 16),             # groups of 3
    ([77], [33], 20, 4, 64, 16),              # groups of 5
    ([700], [203], 64, 4, 128, 16),
    ([0], [515], 32, 4, 128, 16),
    ([3000], [64], 128, 1, 64, 16),           # a group wider than a tile
    ([100, 0, 0, 900, 30], [1, 40, 1, 7, 130], 32, 4, 128, 16),
    ([40, 10, 9, 0], [0, 3, 0, 1], 16, 2, 64, 16),  # sequences without rows
    ([0] * 40 + [512] * 24, [1] * 40 + [2] * 24, 8, 8, 64, 16),
    ([3] * 130, [1, 2] * 65, 4, 2, 128, 16),  # more sequences than lanes
    ([9000, 4000], [40, 1], 24, 3, 64, 16),   # three kv heads: 255 workgroups
    ([2500, 0, 700], [700, 90, 1], 12, 6, 128, 80),
]


@pytest.mark.parametrize("q_f16", [False, True])
@pytest.mark.parametrize("ctx_lens,new,hq,hkv,d,page", ATTENTION)
def test_paged_attention(ctx, hip, ctx_lens, new, hq, hkv, d, page, q_f16):
    print(f"[paged_attention] ctx={ctx_lens[:8]} new={new[:8]} {hq}/{hkv}x{d} page={page} f16={q_f16}", flush=True)
    check_attention(ctx, hip, Batch(1, ctx_lens, new, hq, hkv, d, page, behind=3, q_f16=q_f16), q_f16)


def test_paged_attention_many_sequences(ctx, hip):
    g = np.random.default_rng(5)
    check_attention(ctx, hip, Batch(2, g.integers(0, 60, 1024).tolist(), g.integers(0, 3, 1024).tolist(), 4, 1, 64))


@pytest.mark.parametrize("new,q_f16", [(1, False), (33, True)])
def test_paged_attention_long_parts(ctx, hip, new, q_f16):
    """More tiles than workgroups, of 24000 positions each: parts of a tile longer than the 16384 positions
    whose pages a workgroup holds at a time. (Wide and narrow tiles; the sequences share their pages.)"""
    check_attention(ctx, hip, Batch(9, [24000 - 7 * i for i in range(34)], [new] * 34, 8, 8, 64, 48, pool=100, q_f16=q_f16), q_f16)


@pytest.mark.parametrize("std", [1e-3, 30.0])
def test_paged_attention_small_and_large_scores(ctx, hip, std):
    """q and the caches scaled: nearly uniform weights, and weights of one position alone."""
    check_attention(ctx, hip, Batch(3, [500, 3], [1, 40], 16, 2, 128, std=std))


@pytest.mark.parametrize("scale", [0.0, -0.09, 1e-30])
def test_paged_attention_scales(ctx, hip, scale):
    c = Batch(4, [90, 200], [1, 40], 8, 2, 64)
    c.scale = float(np.float32(scale))
    check_attention(ctx, hip, c)


def test_paged_attention_large_q_small_k(ctx, hip):
    """q beyond f16's range against a cache that makes ordinary scores of it."""
    c = Batch(6, [90, 200], [1, 40], 8, 2, 64)
    c.q *= np.float32(3e6)
    c.kp = (c.kp.astype(np.float32) / 1024).astype(np.float16)
    c.scale = float(np.float32(c.scale * 1024 / 3e6))
    check_attention(ctx, hip, c)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_paged_attention_unattended_values(ctx, hip, bad):
    """Values of later positions of the same sequence do not reach earlier rows; rows that attend them show them."""
    c = Batch(7, [70, 20], [40, 3], 8, 2, 64)
    want, tol = c.attention()
    for pool in (c.kp, c.vp):
        pool[:, c.slots(0, 100)[99]] = bad  # position 99: row 29 of sequence 0
    got = run_attention(ctx, hip, c)
    keep = np.r_[0:29, 40:43]
    assert np.all(np.abs(got[keep] - want[keep]) <= tol[keep])
    assert not np.isfinite(got[29:40]).all(axis=(1, 2)).any()
    # a value alone: the rows before it as they were, the rows that attend it infinite or NaN in its element
    c = Batch(7, [70, 20], [40, 3], 8, 2, 64)
    c.vp[1, c.slots(0, 100)[99], 5] = bad
    got = run_attention(ctx, hip, c)
    assert np.all(np.abs(got[keep] - want[keep]) <= tol[keep])
    assert np.all(got[29:40, 4:, 5] == bad) if not np.isnan(bad) else np.isnan(got[29:40, 4:, 5]).all()
    rest = np.delete(got[29:40], 5, axis=2)
    assert np.all(np.abs(rest - np.delete(want[29:40], 5, axis=2)) <= tol[29:40])


def test_paged_attention_bad_entries(ctx, hip):
    """Device-side lengths, starts and pages out of range: NaN in those rows alone."""
    ctx_lens, new = [50, 200, 30, 9, 400, 60], [1, 40, 2, 1, 1, 1]
    c = Batch(8, ctx_lens, new, 8, 2, 64, behind=2)
    want, tol = c.attention()
    c.seq_lens[0] = c.max_len + 1            # longer than the bound
    c.seq_lens[2] = 1                        # shorter than its rows
    c.table[1, 220 // 16] = c.n_pages        # positions 208 .. 223: rows 8 .. of sequence 1
    c.table[4, 2] = -1
    c.starts[6] = c.rows + 1                 # sequence 5's rows leave the batch
    got = run_attention(ctx, hip, c)
    s = [0, 1, 41, 43, 44, 45]
    bad = np.zeros(c.rows, bool)
    bad[0] = bad[s[2]:s[3]] = bad[s[4]] = bad[s[5]:] = True
    bad[s[1] + 8:s[2]] = True
    assert np.isnan(got[bad]).all()
    assert np.all(np.abs(got[~bad] - want[~bad]) <= tol[~bad])
    for starts in ([0, 1, 41, 20, 44, 45, 46], [-3, 1, 41, 43, 44, 45, 46], [2 ** 31 - 1] * 7, [-2 ** 31] * 7):
        c.starts = np.array(starts, np.int32)  # decreasing, negative, out of range: inside the buffers, whatever it writes
        out = dev(ctx, np.full((c.rows + 64, c.hq * c.d), 7.0, np.float32))
        args = hip.PagedAttentionArgs(dev(ctx, c.q), dev(ctx, c.kp), dev(ctx, c.vp), dev(ctx, c.table), dev(ctx, c.starts),
                                      dev(ctx, c.seq_lens), out.view(0, c.rows * c.hq * c.d * 4), *c.shape(hip, False), c.scale)
        hip.pagedAttention(ctx, args)
        assert np.all(ctx.to_numpy(out, np.float32, (c.rows + 64, c.hq * c.d))[c.rows:] == 7.0)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def check_append(ctx, hip, c, q_f16, norms=True, with_q=True, in_place=False, freq_scale=1.0, theta=THETA):
    g = c.g
    q = g.standard_normal((c.rows, c.hq, c.d)).astype(np.float32)
    k, v = (g.standard_normal((c.rows, c.hkv, c.d)).astype(np.float32) for _ in range(2))
    qn, kn = (g.normal(1.0, 0.02, c.d).astype(np.float32) if norms else None for _ in range(2))
    none = hip.Buf()
    fill = np.full((c.rows, c.hq, c.d), 7.0, np.float16 if q_f16 else np.float32)
    qb = dev(ctx, q) if with_q else none
    qo = (qb if in_place else dev(ctx, fill)) if with_q else none
    kb, vb = dev(ctx, c.kp), dev(ctx, c.vp)
    hip.pagedAppend(ctx, hip.PagedAppendArgs(qb, dev(ctx, k), dev(ctx, v), dev(ctx, qn) if norms else none, dev(ctx, kn) if norms else none, qo,
                                             kb, vb, dev(ctx, c.table), dev(ctx, c.starts), dev(ctx, c.seq_lens), *c.shape(hip, q_f16),
                                             EPS, theta, freq_scale))
    wk, wv = c.kp.astype(np.float64), c.vp.copy()
    pos = np.concatenate([[0]] + [np.arange(a, a + n) for a, n in zip(c.ctx, c.new)])[1:]
    slots = np.concatenate([[0]] + [c.slots(b, c.lens[b])[c.ctx[b]:] for b in range(len(c.ctx))])[1:].astype(np.int64)

    # f32: the norm's and the rotation's roundings and the angle's (under 2 pi 2^-25 + an ulp of sine and
    # cosine), each relative to the rotated pair: 20 half steps. f16 adds its own.
    def tol(want, x, w, f16):
        y = turned(x, w, np.zeros(len(x)), theta, EPS)
        mag = np.hypot(y[..., :c.d // 2], y[..., c.d // 2:])
        t = np.concatenate([mag, mag], -1) * 20 * 2.0 ** -24
        return t + np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if f16 else t

    if with_q:
        got = ctx.to_numpy(qo, fill.dtype, fill.shape)
        want = turned(q[:c.T], qn, pos, theta, EPS, freq_scale)
        assert np.all(np.abs(got[:c.T] - want) <= tol(want, q[:c.T], qn, q_f16))
        assert np.array_equal(got[c.T:], (q if in_place else fill)[c.T:])
    gk, gv = (ctx.to_numpy(b, np.float16, c.kp.shape) for b in (kb, vb))
    want = turned(k[:c.T], kn, pos, theta, EPS, freq_scale)
    assert np.all(np.abs(gk[:, slots].transpose(1, 0, 2) - want) <= tol(want, k[:c.T], kn, True))
    wv[:, slots] = v[:c.T].astype(np.float16).transpose(1, 0, 2)
    assert np.array_equal(gv.view(np.uint16), wv.view(np.uint16))
    other = np.ones(c.kp.shape[1], bool)
    other[slots] = False
    assert np.array_equal(gk[:, other].view(np.uint16), c.kp[:, other].view(np.uint16))  # untouched, NaN and all
    return wk


APPEND = [  # ctx, new, hq, hkv, d, page
    ([0], [1], 32, 4, 128, 16),
    ([4095], [1], 32, 4, 128, 16),
    ([15, 16, 17, 31], [1, 1, 1, 2], 8, 2, 64, 16),
    ([100, 0, 7, 0], [0, 33, 1, 0], 20, 4, 64, 48),
    ([0, 1000], [515, 20], 64, 4, 128, 32),
    ([3] * 100, [1, 2] * 50, 4, 2, 128, 16),
    ([1] * 4200, [1] * 4200, 2, 1, 64, 16),
    ([5], [9], 128, 8, 128, 16),              # 144 heads a token
]


@pytest.mark.parametrize("q_f16", [False, True])
@pytest.mark.parametrize("ctx_lens,new,hq,hkv,d,page", APPEND)
def test_paged_append(ctx, hip, ctx_lens, new, hq, hkv, d, page, q_f16):
    print(f"[paged_append] ctx={ctx_lens[:8]} new={new[:8]} {hq}/{hkv}x{d} page={page} f16={q_f16}", flush=True)
    check_append(ctx, hip, Batch(11, ctx_lens, new, hq, hkv, d, page, behind=3), q_f16)


@pytest.mark.parametrize("kw", [dict(norms=False), dict(with_q=False), dict(in_place=True), dict(freq_scale=0.25), dict(theta=1e4)])
def test_paged_append_options(ctx, hip, kw):
    check_append(ctx, hip, Batch(12, [50, 0], [3, 20], 8, 2, 128, behind=2), False, **kw)


def test_paged_append_far_positions(ctx, hip):
    """A long page table: positions up to 2^21, the angle as exact as at the beginning."""
    c = Batch(13, [0, 0], [2, 3], 4, 2, 128, page=16)
    far = [131072 - 2, 2 ** 21 - 3]
    c.max_pages = 2 ** 21 // 16
    table = np.full((2, c.max_pages), -7, np.int32)
    for b in range(2):
        table[b, far[b] // 16:(far[b] + 3 + 15) // 16] = c.table[b, 0]
    c.ctx, c.table, c.max_len = far, table, 2 ** 21
    c.lens = [a + n for a, n in zip(c.ctx, c.new)]
    c.seq_lens = np.array(c.lens, np.int32)
    check_append(ctx, hip, c, False)


def test_paged_append_bad_entries(ctx, hip):
    c = Batch(14, [50, 20, 30], [2, 2, 17], 4, 2, 64, behind=1)
    ok = c.table.copy()
    c.seq_lens[0] = 1
    c.table[1, 1] = c.n_pages           # the page of both rows of sequence 1
    c.table[2, 2] = -1                  # positions 32 .. 46: row 2 on
    g = c.g
    q, k, v = (g.standard_normal((c.rows, h, c.d)).astype(np.float32) for h in (4, 2, 2))
    none, kb, vb, qb = hip.Buf(), dev(ctx, c.kp), dev(ctx, c.vp), dev(ctx, q)
    hip.pagedAppend(ctx, hip.PagedAppendArgs(qb, dev(ctx, k), dev(ctx, v), none, none, qb, kb, vb, dev(ctx, c.table), dev(ctx, c.starts),
                                             dev(ctx, c.seq_lens), *c.shape(hip, False), EPS, THETA, 1.0))
    got = ctx.to_numpy(qb, np.float32, q.shape)
    assert np.isnan(got[:4]).all() and np.isfinite(got[4:6]).all() and np.isnan(got[6:21]).all() and np.array_equal(got[21:], q[21:])
    gv = ctx.to_numpy(vb, np.float16, c.vp.shape)
    want = c.vp.copy()
    s = [int(ok[2, p // 16]) * 16 + p % 16 for p in (30, 31)]
    want[:, s] = v[4:6].astype(np.float16).transpose(1, 0, 2)
    assert np.array_equal(gv.view(np.uint16), want.view(np.uint16))


def test_append_attention_graph(ctx, hip):
    """Both captured once and replayed as the sequences grow: each replay as the eager calls, bit for bit."""
    c = Batch(15, [30, 500, 0], [1, 1, 1], 16, 2, 128, spare=8)
    c.table[:] = np.arange(3 * c.max_pages).reshape(3, -1) % c.n_pages
    c.max_len = c.max_pages * 16
    need = 3 * c.max_pages
    c.n_pages = need
    c.table[:] = np.random.default_rng(1).permutation(need).reshape(3, -1)
    pool = np.random.default_rng(2).standard_normal((2, 2, need * 16, 128)).astype(np.float16)
    q, k, v = (c.g.standard_normal((3, h, 128)).astype(np.float32) for h in (16, 2, 2))
    qb, kb, vb = dev(ctx, q), dev(ctx, k), dev(ctx, v)
    outs = []
    for graph in (False, True):
        qo, out = ctx.createBuffer(q.nbytes), ctx.createBuffer(q.nbytes)
        kp, vp, lens = dev(ctx, pool[0]), dev(ctx, pool[1]), dev(ctx, c.seq_lens)
        tail = (kp, vp, dev(ctx, c.table), dev(ctx, c.starts), lens)
        none = hip.Buf()
        aa = hip.PagedAppendArgs(qb, kb, vb, none, none, qo, *tail, *c.shape(hip, False), EPS, THETA, 1.0)
        at = hip.PagedAttentionArgs(qo, *tail, out, *c.shape(hip, False), c.scale)

        def both():
            hip.pagedAppend(ctx, aa)
            hip.pagedAttention(ctx, at)

        g = ctx.capture(both) if graph else None
        got = []
        for i in range(4):
            ctx.upload(lens, 0, c.seq_lens + np.int32(i))
            ctx.upload(qb, 0, q + np.float32(i))
            g.launch() if graph else both()
            got.append((ctx.to_numpy(out, np.uint32), ctx.to_numpy(kp, np.uint16), ctx.to_numpy(vp, np.uint16)))
        if graph:
            g.destroy()
        outs.append(got)
    for a, b in zip(*outs):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))
    assert not np.array_equal(outs[0][0][0], outs[0][3][0])


@pytest.mark.parametrize("d,q_f16", [(128, False), (128, True), (64, False), (64, True)])
def test_paged_attention_wide_tiles_again(ctx, hip, d, q_f16):
    """Wide tiles of odd and even counts of 64-position steps, whole and cut, 40 times: right, and the same bits."""
    c = Batch(22, [0, 1, 90, 150, 217, 281, 3000], [64, 130, 40, 41, 39, 300, 70], 16, 2, d, q_f16=q_f16)
    check_attention(ctx, hip, c, q_f16)
    want = run_attention(ctx, hip, c, q_f16)
    for _ in range(20):
        assert np.array_equal(run_attention(ctx, hip, c, q_f16).view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("new,d,q_f16", [(1, 128, False), (1, 64, True), (40, 128, True), (40, 64, False)])
def test_paged_attention_keys_of_nan(ctx, hip, new, d, q_f16):
    """NaN in every key of a span that ends, at one of the ends tried, where a part of the cut tile does: parts that hold
    nothing else make the rows that attend them NaN all the same. The other kv head's rows, and another sequence's,
    are as they were."""
    c = Batch(21, [4000 - new, 50], [new, 1], 16, 2, d, q_f16=q_f16)
    want, tol = c.attention()
    tol = np.broadcast_to(tol, want.shape)
    slots, kp = c.slots(0, 4000), c.kp.copy()
    for end in [*range(64, 2048, 64), 4000]:
        c.kp[1, slots[:end]] = np.nan
        got = run_attention(ctx, hip, c, q_f16)
        assert np.isnan(got[:new, 8:]).all(), end
        err = np.abs(got - want)
        assert np.all(err[:new, :8] <= tol[:new, :8]) and np.all(err[new:] <= tol[new:])
        c.kp[:] = kp


@pytest.mark.parametrize("q_f16", [False, True])
def test_paged_attention_scale_of_nan(ctx, hip, q_f16):
    c = Batch(23, [5000, 90], [1, 40], 8, 2, 64, q_f16=q_f16)
    assert np.isnan(run_attention(ctx, hip, c, q_f16, scale=float("nan"))).all()


def test_paged_attention_huge_q_tiny_scale(ctx, hip):
    """A scale below the normal floats, of q near the largest: ordinary scores."""
    c = Batch(24, [900, 200], [1, 40], 8, 2, 64)
    c.q *= np.float32(3e37)
    c.scale = float(np.float32(c.scale / 3e37))
    check_attention(ctx, hip, c)


@pytest.mark.parametrize("bits", [6, 11, 16, 22, 28, 34])
@pytest.mark.parametrize("seqs,new", [(1, 1), (64, 1), (1, 40), (64, 20)])
def test_paged_attention_flat_tail(ctx, hip, seqs, new, bits):
    """One dominant position, of value 0, before 2^15 of equal weights 2^-bits of its own, of value 1: the weights' 22
    bits, or 2^-33 of the dominant one, are what the sum over the tail may be off by. (64 sequences of the same
    pages: whole tiles; one: cut.)"""
    hq, hkv, d, L = 16, 4, 64, 2 ** 15
    score = np.float32(bits * np.log(2.0))
    q = np.zeros((seqs * new, hq, d), np.float32)
    q[..., 0] = score
    kp, vp = np.zeros((hkv, L, d), np.float16), np.ones((hkv, L, d), np.float16)
    kp[:, 0, 0], vp[:, 0] = 8, 0
    table = np.tile(np.arange(L // 16, dtype=np.int32), (seqs, 1))
    out = ctx.createBuffer(q.nbytes)
    hip.pagedAttention(ctx, hip.PagedAttentionArgs(
        dev(ctx, q), dev(ctx, kp), dev(ctx, vp), dev(ctx, table), dev(ctx, np.arange(seqs + 1, dtype=np.int32) * np.int32(new)),
        dev(ctx, np.full(seqs, L, np.int32)), out, hip.DTYPE_F32, seqs * new, seqs, hq, hkv, d, 16, L // 16, L // 16, L, 0.125))
    got = ctx.to_numpy(out, np.float32, (seqs, new, hq * d))
    tail = np.arange(L - new, L)[None, :, None].astype(np.float64) * np.exp(-np.float64(score))
    want = tail / (1 + tail)
    # relative: the score's 22 bits and its roundings in log2 units (3 half steps), the weight's 22 bits and its own
    # rounding, and the sums', 16 positions a step; a weight's sum is of the unsplit weights, so that both count once
    rel = 2.0 ** -22 * float(score) + bits * 3 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -23 + 2 * (L / 16 + 64) * 2.0 ** -24
    assert np.all(np.abs(got - want) <= want * rel + L * 2.0 ** -33 / (1 + tail)), float(np.abs(got - want).max())


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("bits", [8, 16, 20])
def test_paged_attention_q_with_one_large_element(ctx, hip, new, bits):
    """Elements of an f32 q beside one 2^bits as large, which meets zeros of K: 22 bits of each, or 2^-38 of the largest."""
    c = Batch(25, [900], [new], 8, 2, 64)
    c.q[..., 0] = np.ldexp(1.5, bits) * np.sign(c.q[..., 0])
    c.kp[..., 0] = 0
    want, tol = c.attention()
    delta = c.scale * np.abs(np.nan_to_num(c.kp.astype(np.float64))).sum(-1).max() * 2.0 ** -38 * np.ldexp(1.5, bits)
    got = run_attention(ctx, hip, c)
    # a score off by delta moves its weight by as much of itself, and the weights' sum by as much again
    assert np.all(np.abs(got - want) <= tol + 2 * delta * np.nanmax(np.abs(c.vp.astype(np.float64))))


def test_paged_append_refused_rows_write_nothing(ctx, hip):
    """Neither pool changes but in the slots of the rows that are in range, with q and without."""
    for with_q in (True, False):
        c = Batch(26, [50, 20, 30], [2, 2, 17], 4, 2, 64, behind=1)
        slots = c.slots(2, 32)[30:]         # positions 30 and 31 of sequence 2: the rows that are whole
        c.seq_lens[0] = 1
        c.table[1, 1] = c.n_pages           # the page of both rows of sequence 1
        c.table[2, 2] = -1                  # positions 32 .. 46
        q, k, v = (c.g.standard_normal((c.rows, h, c.d)).astype(np.float32) for h in (4, 2, 2))
        none, kb, vb, qb = hip.Buf(), dev(ctx, c.kp), dev(ctx, c.vp), dev(ctx, q)
        hip.pagedAppend(ctx, hip.PagedAppendArgs(qb if with_q else none, dev(ctx, k), dev(ctx, v), none, none, qb if with_q else none, kb, vb,
                                                 dev(ctx, c.table), dev(ctx, c.starts), dev(ctx, c.seq_lens), *c.shape(hip, False), EPS, THETA, 1.0))
        for b, was in ((kb, c.kp), (vb, c.vp)):
            got = ctx.to_numpy(b, np.uint16, was.shape)
            same = (got == was.view(np.uint16)).all(axis=(0, 2))
            assert sorted(np.flatnonzero(~same)) == sorted(slots.tolist())
        # f32: the rotation's roundings, 20 half steps of the pair at most; f16 its own half step
        want = turned(k[4:6], None, [30, 31], THETA, EPS)
        mag = np.hypot(k[4:6, :, :32], k[4:6, :, 32:])
        got = ctx.to_numpy(kb, np.float16, c.kp.shape)[:, slots].transpose(1, 0, 2)
        assert np.all(np.abs(got - want) <= np.concatenate([mag, mag], -1) * 20 * 2.0 ** -24 + np.abs(want) * 2.0 ** -11 + 2.0 ** -25)
